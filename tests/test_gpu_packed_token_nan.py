"""Tokens against a long cache whose keys are split over workgroups: a NaN that a token sees stays a NaN, one that is hidden
from it reaches nothing, however many of a split's scores are NaN."""
import math

import pytest
import torch

from tests.packed_reference import check, reference

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.float16, torch.bfloat16]
SHAPES = [(8, 5, 5), (64, 4, 2), (128, 8, 1)]


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _case(dtype, dim, heads, kv, lengths, bias):
    import imageni2r_amd as i2r
    gen = torch.Generator(DEV).manual_seed(dim + len(lengths))
    room, batch = max(lengths), len(lengths)
    rand = lambda *s: torch.randn(*s, generator=gen, device=DEV).to(dtype)
    q, k, v = rand(batch, heads, dim), rand(batch * room, kv, dim), rand(batch * room, kv, dim)
    buckets = i2r.RelativeBuckets(16, 64, False) if bias else None
    table = torch.randn(heads, 16, generator=gen, device=DEV) if bias else None
    at = [room * b for b in range(batch + 1)]
    seqs = i2r.PackedSequences(_i32(list(range(batch + 1))), _i32(at), len_k=_i32(lengths), causal=True, buckets=buckets)
    return q, k, v, table, seqs, dict(cu_q=list(range(batch + 1)), cu_k=at, len_k=lengths, causal=True, table=table,
                                      buckets=buckets)


def _splits(q, k, seqs):
    """Whether the call splits its keys (it needs a workspace then)."""
    from imageni2r_amd import _lib, packed
    return _lib.query("i2r_packed_attention_fwd_ws_bytes", packed._DTYPES[q.dtype], seqs.batch, q.shape[0], k.shape[0],
                      q.shape[1], k.shape[1], q.shape[2]) > 0


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dim,heads,kv", SHAPES)
@pytest.mark.parametrize("bias", [False, True], ids=["plain", "bias"])
@pytest.mark.parametrize("lengths", [[40], [5000], [5000, 1, 2600, 4999]], ids=str)
def test_a_token_that_is_nan(dtype, dim, heads, kv, bias, lengths):
    import imageni2r_amd as i2r
    q, k, v, table, seqs, ref = _case(dtype, dim, heads, kv, lengths, bias)
    assert _splits(q, k, seqs) == (max(lengths) > 1000)
    want = reference(q, k, v, **ref)["out"]
    q[-1, heads - 1, 3] = math.nan
    got = i2r.packed_attention(q, k, v, seqs, bias=table)
    assert bool(torch.isnan(got[-1, heads - 1]).all())
    clean = torch.ones(q.shape[:2], dtype=torch.bool, device=DEV)
    clean[-1, heads - 1] = False
    check("out", got[clean], want[0][clean], want[1][clean])
    # the backward reads what the forward kept: the row's gradient is NaN too
    leaf = q.clone().requires_grad_(True)
    dq = torch.autograd.grad(i2r.packed_attention(leaf, k, v, seqs, bias=table).float().sum(), leaf)[0]
    assert bool(torch.isnan(dq[-1, heads - 1]).all()) and bool(torch.isfinite(dq[clean]).all())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dim,heads,kv", SHAPES)
@pytest.mark.parametrize("bias", [False, True], ids=["plain", "bias"])
def test_a_whole_split_of_nan_keys(dtype, dim, heads, kv, bias):
    """Six of a sequence's splits (of 256 keys each) hold nothing but NaN.  Its token is NaN, the other's values right."""
    import imageni2r_amd as i2r
    q, k, v, table, seqs, ref = _case(dtype, dim, heads, kv, [4096, 4096], bias)
    assert _splits(q, k, seqs)
    want = reference(q, k, v, **ref)["out"]
    k[1024:2560] = math.nan
    got = i2r.packed_attention(q, k, v, seqs, bias=table)
    assert bool(torch.isnan(got[0]).all())
    check("out", got[1], want[0][1], want[1][1])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dim,heads,kv", SHAPES)
def test_splits_of_nan_that_are_hidden(dtype, dim, heads, kv):
    """The bucket of all keys 64 and more steps back is -inf, and those keys are NaN: the tokens see the others alone."""
    import imageni2r_amd as i2r
    q, k, v, table, seqs, ref = _case(dtype, dim, heads, kv, [5000, 4000], True)
    table[:, 15] = -math.inf
    want = reference(q, k, v, **ref)["out"]
    k[:4900], v[:4900], k[5000:8900], v[5000:8900] = math.nan, math.inf, math.inf, math.nan
    check("out", i2r.packed_attention(q, k, v, seqs, bias=table), *want)
