"""Attention over packed sequences (imageni2r_amd.packed) against its formulas in 64 bits."""
import math

import pytest
import torch

from tests.packed_reference import check, reference

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _cu(lengths, first=0):
    cu = [first]
    for n in lengths:
        cu.append(cu[-1] + n)
    return cu


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _rand(gen, *shape, dtype=F32, size=1.0):
    return (torch.randn(*shape, generator=gen, device=DEV) * size).to(dtype)


def _make(gen, dtype, dim, heads, kv, lens_q, lens_k=None, bias=None, positions=False, causal=False, fused=False):
    import imageni2r_amd as i2r
    cu_q, cu_k = _cu(lens_q), None if lens_k is None else _cu(lens_k)
    nq, nk = cu_q[-1], cu_q[-1] if cu_k is None else cu_k[-1]
    if fused:
        qkv = _rand(gen, nq, heads + 2 * kv, dim, dtype=dtype)
        q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    else:
        q, k, v = _rand(gen, nq, heads, dim, dtype=dtype), _rand(gen, nk, kv, dim, dtype=dtype), \
            _rand(gen, nk, kv, dim, dtype=dtype)
    buckets = table = pos_q = pos_k = None
    if bias:
        buckets = i2r.RelativeBuckets(*bias)
        table = _rand(gen, heads, bias[0])
    if positions:
        pos_q = torch.randint(0, 300, (nq,), generator=gen, device=DEV).int()
        pos_k = None if cu_k is None else torch.randint(0, 300, (nk,), generator=gen, device=DEV).int()
    seqs = i2r.PackedSequences(_i32(cu_q), None if cu_k is None else _i32(cu_k), causal=causal, buckets=buckets,
                               pos_q=pos_q, pos_k=pos_k)
    ref = dict(cu_q=cu_q, cu_k=cu_k, causal=causal, table=table, buckets=buckets, pos_q=pos_q, pos_k=pos_k)
    return q, k, v, table, seqs, ref


def _grads(q, k, v, table, seqs, dout, scale=None):
    import imageni2r_amd as i2r
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    t = None if table is None else table.detach().clone().requires_grad_(True)
    out = i2r.packed_attention(*leaves, seqs, bias=t, scale=scale)
    got = torch.autograd.grad(out, leaves + ([] if t is None else [t]), dout)
    return dict(zip(("out", "dq", "dk", "dv", "dtable"), (out.detach(),) + got))


def _all(gen, q, k, v, table, seqs, ref, scale=None):
    import imageni2r_amd as i2r
    dout = _rand(gen, *q.shape, dtype=q.dtype)
    want = reference(q, k, v, scale=scale, dout=dout, **ref)
    with torch.no_grad():
        check("out, inference", i2r.packed_attention(q, k, v, seqs, bias=table, scale=scale), *want["out"])
    got = _grads(q, k, v, table, seqs, dout, scale)
    for name, w in want.items():
        check(name, got[name], *w)


RAGGED = [1, 17, 64, 0, 130, 3, 255]


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,heads,kv", [(8, 5, 5), (32, 2, 1), (40, 3, 3), (64, 6, 2), (72, 4, 1), (128, 4, 2), (96, 2, 2)])
@pytest.mark.parametrize("causal", [False, True], ids=["both", "causal"])
def test_ragged_sequences(dtype, dim, heads, kv, causal):
    gen = torch.Generator(DEV).manual_seed(dim + heads)
    _all(gen, *_make(gen, dtype, dim, heads, kv, RAGGED, causal=causal, fused=True))


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("bias", [(32, 128, True), (8, 20, True), (64, 1024, False), (6, 9, False)], ids=str)
@pytest.mark.parametrize("causal,positions", [(False, False), (False, True), (True, False), (True, True)])
@pytest.mark.parametrize("dim,heads,kv", [(8, 5, 5), (64, 4, 2), (128, 2, 1)])
def test_bias(dtype, bias, causal, positions, dim, heads, kv):
    gen = torch.Generator(DEV).manual_seed(bias[0] + dim)
    _all(gen, *_make(gen, dtype, dim, heads, kv, [1, 200, 0, 33, 300], bias=bias, positions=positions, causal=causal))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("dim,heads,kv", [(16, 4, 4), (64, 8, 1), (128, 6, 2)])
@pytest.mark.parametrize("bias", [None, (16, 50, False)], ids=["plain", "bias"])
def test_other_keys_than_queries(dtype, dim, heads, kv, bias):
    """Cross lengths, causal: more keys, fewer keys (rows that see nothing), none, and queries of no length."""
    gen = torch.Generator(DEV).manual_seed(3)
    case = _make(gen, dtype, dim, heads, kv, [5, 40, 70, 0, 3, 1], [90, 33, 0, 12, 130, 1], bias=bias, causal=True)
    _all(gen, *case)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 3])
@pytest.mark.parametrize("dim,heads,kv", [(64, 8, 8), (128, 16, 2), (80, 12, 3), (8, 5, 5)])
@pytest.mark.parametrize("bias", [None, (32, 128, False)], ids=["plain", "bias"])
def test_tokens_against_a_cache(dtype, rows, dim, heads, kv, bias):
    import imageni2r_amd as i2r
    gen = torch.Generator(DEV).manual_seed(dim + rows)
    fill, room = [1, 700, 0, 64, 2049, 3000, 65], 3001
    q = _rand(gen, rows * len(fill), heads, dim, dtype=dtype)
    k, v = (_rand(gen, len(fill), room, kv, dim, dtype=dtype) for _ in range(2))
    for b, n in enumerate(fill):  # what lies behind the fill is never used
        k[b, n:], v[b, n:] = math.nan, math.inf
    buckets = i2r.RelativeBuckets(*bias) if bias else None
    table = _rand(gen, heads, bias[0]) if bias else None
    cu_q, cu_k = [rows * b for b in range(len(fill) + 1)], [room * b for b in range(len(fill) + 1)]
    seqs = i2r.PackedSequences(_i32(cu_q), _i32(cu_k), len_k=_i32(fill), causal=True, buckets=buckets)
    k, v = k.view(-1, kv, dim), v.view(-1, kv, dim)
    want = reference(q, k, v, cu_q, cu_k, fill, True, table=table, buckets=buckets)
    check("out", i2r.packed_attention(q, k, v, seqs, bias=table), *want["out"])
    seqs.len_k.copy_(_i32([n + 1 for n in fill]))  # the fill is read when the kernel runs
    k, v = torch.nan_to_num(k, 0.5, 0.5), torch.nan_to_num(v, 0.5, 0.5, 0.5)
    want = reference(q, k, v, cu_q, cu_k, [n + 1 for n in fill], True, table=table, buckets=buckets)
    check("out of the longer cache", i2r.packed_attention(q, k, v, seqs, bias=table), *want["out"])


@pytest.mark.parametrize("dtype", [F16, BF16, F32], ids=["f16", "bf16", "f32"])
@pytest.mark.parametrize("causal", [False, True])
def test_long_sequences(dtype, causal):
    gen = torch.Generator(DEV).manual_seed(1)
    _all(gen, *_make(gen, dtype, 64, 2, 1, [2500, 1, 1031], bias=(32, 128, False), causal=causal))


def test_one_token_alone_and_one_row():
    gen = torch.Generator(DEV).manual_seed(1)
    for dtype in (F32, F16, BF16):
        q, k, v, table, seqs, ref = _make(gen, dtype, 64, 4, 2, [1])
        import imageni2r_amd as i2r
        assert torch.equal(i2r.packed_attention(q, k, v, seqs), v.repeat_interleave(2, 1))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("dim", [8, 64, 128])
def test_rows_of_no_sequence(dtype, dim):
    """Rows before the first and behind the last sequence, and keys behind a fill: left as they were with out=, zero
    without, and so are their gradients; what they hold (NaN here) reaches nothing."""
    import imageni2r_amd as i2r
    gen = torch.Generator(DEV).manual_seed(9)
    lens, first, n = [40, 0, 150], 37, 300
    cu = _cu(lens, first)
    q, k, v, dout = (_rand(gen, n, 2, dim, dtype=dtype) for _ in range(4))
    for t in (q, k, v, dout):
        t[:first], t[cu[-1]:] = math.nan, math.nan
    fill = [30, 0, 150]
    k[first + 30:first + 40], v[first + 30:first + 40] = math.inf, math.nan
    seqs = i2r.PackedSequences(_i32(cu), _i32(cu), len_k=_i32(fill))
    want = reference(q, k, v, cu, cu, fill, dout=dout)
    got = _grads(q, k, v, None, seqs, dout)
    for name, w in want.items():
        check(name, got[name], *w)
        assert bool((got[name][:first] == 0).all()) and bool((got[name][cu[-1]:] == 0).all()), name
    mark = torch.full_like(q, 7.0)
    assert i2r.packed_attention(q, k, v, seqs, out=mark) is mark
    assert bool((mark[:first] == 7).all()) and bool((mark[cu[-1]:] == 7).all())
    check("out=", mark[first:cu[-1]], want["out"][0][first:cu[-1]], want["out"][1][first:cu[-1]])


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,heads,kv", [(16, 2, 1), (64, 2, 1), (128, 2, 1), (64, 2, 2), (128, 2, 2), (96, 128, 64)])
def test_hidden_values_are_never_used(dtype, dim, heads, kv):
    """Causal: NaN and infinities in a sequence's last key and value row reach its last query alone, forward and
    backward; the last query's own NaN gradient reaches what it sees, but no earlier row's dq."""
    import imageni2r_amd as i2r
    gen = torch.Generator(DEV).manual_seed(dim)
    lens = [70, 1, 129]
    q, k, v, _, seqs, ref = _make(gen, dtype, dim, heads, kv, lens, causal=True)
    clean = reference(q, k, v, dout=(dout := _rand(gen, *q.shape, dtype=dtype)), **ref)
    ends = [n - 1 for n in _cu(lens)[1:]]
    for bad_k, bad_v in ((math.nan, math.nan), (math.inf, -math.inf), (1.0, math.nan)):
        k2, v2 = k.clone(), v.clone()
        k2[ends], v2[ends] = bad_k, bad_v
        keep = torch.ones(q.shape[0], dtype=torch.bool, device=DEV)
        keep[ends] = False
        out = i2r.packed_attention(q, k2, v2, seqs)
        check("out", out[keep], clean["out"][0][keep], clean["out"][1][keep])
        assert bool(torch.isnan(out[ends].float()).any(-1).all())
        got = _grads(q, k2, v2, None, seqs, dout)
        check("dq", got["dq"][keep], clean["dq"][0][keep], clean["dq"][1][keep])
    dout[ends] = math.nan
    got = _grads(q, k, v, None, seqs, dout)
    check("dq", got["dq"][keep], clean["dq"][0][keep], clean["dq"][1][keep])
    # a later query's NaN does not reach the keys that it cannot see
    first = [_cu(lens)[0], _cu(lens)[2]]
    q2, dout2 = q.clone(), _rand(gen, *q.shape, dtype=dtype)
    want = reference(q, k, v, dout=dout2, **ref)
    q2[first], dout2b = math.nan, dout2.clone()
    dout2b[first] = math.nan
    got = _grads(q2, k, v, None, seqs, dout2b)
    later = torch.ones(q.shape[0], dtype=torch.bool, device=DEV)
    later[first] = False
    for name in ("out", "dq", "dk", "dv"):
        check(name, got[name][later], want[name][0][later], want[name][1][later])


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("positions", [False, True])
def test_table_of_minus_infinity_and_of_the_lowest_value(dtype, positions):
    """-inf buckets hide their keys (rows that see nothing are 0, hidden NaN stay out); the lowest finite value ranks
    keys below all others, and a row that has nothing else weighs them alike."""
    import imageni2r_amd as i2r
    gen = torch.Generator(DEV).manual_seed(4)
    q, k, v, table, seqs, ref = _make(gen, dtype, 64, 3, 3, [150, 40], bias=(16, 40, True), positions=positions)
    table[0] = -math.inf          # head 0 sees nothing
    table[1, 8:] = -math.inf      # head 1 sees only what is behind
    table[2, 3:] = torch.finfo(F32).min
    _all(gen, q, k, v, table, seqs, ref)
    out = i2r.packed_attention(q, k, v, seqs, bias=table)
    assert bool((out[:, 0] == 0).all())
    table[:] = torch.finfo(F32).min
    _all(gen, q, k, v, table, seqs, ref)
    if not positions:  # a key that -inf buckets hide from all queries but its own and later ones
        table[:] = 0.0
        table[:, 9:] = -math.inf
        want = reference(q, k, v, **ref)
        v2 = v.clone()
        v2[149], v2[189] = math.nan, math.inf
        out = i2r.packed_attention(q, k, v2, seqs, bias=table)
        keep = torch.ones(190, dtype=torch.bool, device=DEV)
        keep[[149, 189]] = False
        check("out", out[keep], want["out"][0][keep], want["out"][1][keep])


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
def test_large_and_small_scores(dtype):
    gen = torch.Generator(DEV).manual_seed(6)
    q, k, v, table, seqs, ref = _make(gen, dtype, 64, 2, 2, [100, 90], bias=(8, 20, True))
    for scale in (4.0, 0.0, 1e-4, -0.5):
        _all(gen, q, k, v, table * 30, seqs, dict(ref, table=table * 30), scale)


def test_positions_at_the_ends_of_their_type():
    gen = torch.Generator(DEV).manual_seed(6)
    q, k, v, table, seqs, ref = _make(gen, F32, 16, 2, 2, [70], bias=(8, 20, True), positions=True)
    ends = _i32([-2**31, 2**31 - 1, 0, -1, 2**31 - 2])
    seqs.pos_q.copy_(ends[torch.randint(0, 5, (70,), generator=gen, device=DEV)])
    _all(gen, q, k, v, table, seqs, ref)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_layouts(dtype):
    """Heads before rows, expanded heads, rows that are not 16-byte aligned: the same values as contiguous operands."""
    import imageni2r_amd as i2r
    gen = torch.Generator(DEV).manual_seed(5)
    q, k, v, _, seqs, ref = _make(gen, dtype, 24, 4, 4, [77, 30], causal=True)
    dout = _rand(gen, *q.shape, dtype=dtype)
    want = _grads(q, k, v, None, seqs, dout)
    t = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
    wide = [torch.zeros(107, 4, 27, dtype=dtype, device=DEV)[..., 3:] for _ in range(3)]
    for w, x in zip(wide, (q, k, v)):
        w.copy_(x)
    for ops in (t, wide):
        got = _grads(*ops, None, seqs, dout.transpose(0, 1).contiguous().transpose(0, 1))
        for n in want:
            assert torch.equal(got[n], want[n]), n
    one = k[:, :1].expand(-1, 4, -1)
    leaf = k[:, :1].detach().clone().requires_grad_(True)
    out = i2r.packed_attention(q, leaf.expand(-1, 4, -1), leaf.expand(-1, 4, -1), seqs)
    assert torch.equal(out, i2r.packed_attention(q, one.contiguous(), one.contiguous(), seqs))
    (g,) = torch.autograd.grad(out, leaf, dout)
    ref1 = reference(q, k[:, :1], k[:, :1], ref["cu_q"], causal=True, dout=dout)
    # broadcast over four heads: four rounded gradients of k and four of v are added
    four = reference(q, one, one, ref["cu_q"], causal=True, dout=dout)
    slack = (four["dk"][1] + four["dv"][1]).sum(1, keepdim=True) + torch.finfo(dtype).eps * 8 * (
        four["dk"][0].abs() + four["dv"][0].abs()).sum(1, keepdim=True)
    check("gradient of a broadcast key", g, ref1["dk"][0] + ref1["dv"][0], slack)


def test_offsets_past_32_bits():
    """A cache whose last rows lie more than 2^32 bytes behind its first."""
    import imageni2r_amd as i2r
    gen = torch.Generator(DEV).manual_seed(5)
    rows, kv, dim = (1 << 21) + 500, 8, 128
    k = torch.empty(rows, kv, dim, dtype=BF16, device=DEV)
    v = torch.empty_like(k)
    k[-400:], v[-400:] = (_rand(gen, 400, kv, dim, dtype=BF16) for _ in range(2))
    q = _rand(gen, 1, kv, dim, dtype=BF16)
    seqs = i2r.PackedSequences(_i32([0, 1]), _i32([rows - 400, rows]))
    want = reference(q, k[-400:], v[-400:], [0, 1], [0, 400])
    check("out", i2r.packed_attention(q, k, v, seqs), *want["out"])
    q = _rand(gen, 200, kv, dim, dtype=BF16)
    seqs = i2r.PackedSequences(_i32([0, 200]), _i32([rows - 400, rows]), causal=True)
    want = reference(q, k[-400:], v[-400:], [0, 200], [0, 400], causal=True)
    check("out", i2r.packed_attention(q, k, v, seqs), *want["out"])


def test_index_values_outside_the_tensors_are_clamped():
    """Nothing on the host reads the arrays: starts before the first and ends behind the last row mean those rows."""
    import imageni2r_amd as i2r
    gen = torch.Generator(DEV).manual_seed(2)
    for dtype in (F32, BF16):
        q, k, v, _, _, _ = _make(gen, dtype, 64, 2, 2, [100])
        dout = _rand(gen, *q.shape, dtype=dtype)
        good = _grads(q, k, v, None, i2r.PackedSequences(_i32([0, 60, 100])), dout)
        bad = _grads(q, k, v, None, i2r.PackedSequences(_i32([-5, 60, 2**31 - 1]), len_k=_i32([1000, 2**31 - 1])), dout)
        for n in good:
            assert torch.equal(good[n], bad[n]), n


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_the_same_inputs_give_the_same_bits(dtype):
    gen = torch.Generator(DEV).manual_seed(2)
    q, k, v, table, seqs, _ = _make(gen, dtype, 64, 4, 2, [300, 511, 2], bias=(32, 128, True), positions=True)
    dout = _rand(gen, *q.shape, dtype=dtype)
    a = _grads(q, k, v, table, seqs, dout)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        b = _grads(q, k, v, table, seqs, dout)
        with torch.cuda.stream(side):  # and beside the same on another stream
            c = _grads(q, k, v, table, seqs, dout)
        side.synchronize()
        for n in a:
            assert torch.equal(a[n], b[n]) and torch.equal(a[n], c[n]), n


def test_gradients_against_differences():
    """Central differences of the kernel's own forward in fp32: with steps of 2^-6 the truncation is third order
    (2^-12 / 6 times the third derivative, about 1 here) and the loss' rounding 2^-24 * |loss| / step."""
    import imageni2r_amd as i2r
    gen = torch.Generator(DEV).manual_seed(8)
    q, k, v, table, seqs, _ = _make(gen, F32, 8, 2, 1, [9, 14], bias=(8, 6, True), causal=False)
    dout = _rand(gen, *q.shape)
    got = _grads(q, k, v, table, seqs, dout)
    for name, t in (("dq", q), ("dk", k), ("dv", v), ("dtable", table)):
        way = _rand(gen, *t.shape)
        way /= way.norm()
        step, loss = 2.0**-6, []
        for sign in (1, -1):
            moved = {"dq": q, "dk": k, "dv": v, "dtable": table}
            moved[name] = t + sign * step * way
            out = i2r.packed_attention(moved["dq"], moved["dk"], moved["dv"], seqs, bias=moved["dtable"])
            loss.append((out.double() * dout.double()).sum().item())
        slope = (loss[0] - loss[1]) / (2 * step)
        want = (got[name].double() * way.double()).sum().item()
        size = float(dout.double().norm() * v.double().norm())
        assert abs(slope - want) <= size * (2.0**-12 + 2.0**-24 / step), (name, slope, want)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_captured_and_replayed_with_other_lengths(dtype):
    """Two graphs over the same tensors, forward with gradients and a token against a cache; between the replays eager
    work of the same operator, other lengths and other inputs."""
    import imageni2r_amd as i2r
    from imageni2r_amd import packed
    gen = torch.Generator(DEV).manual_seed(3)
    q, k, v, table, seqs, ref = _make(gen, dtype, 64, 4, 2, [100, 60, 90], bias=(16, 40, False), causal=True)
    dout, tok = _rand(gen, *q.shape, dtype=dtype), _rand(gen, 2, 4, 64, dtype=dtype)
    cache = i2r.PackedSequences(_i32([0, 1, 2]), _i32([0, 125, 250]), len_k=_i32([3, 7]), causal=True)

    def train():
        out, out32, stats = packed.packed_attention_fwd(q, k, v, seqs, table, save=True)
        return (out,) + packed.packed_attention_bwd(q, k, v, seqs, table, out32, stats, dout)

    def token():
        return (i2r.packed_attention(tok, k, v, cache),)

    train(), token()
    torch.cuda.synchronize()
    graphs = []
    for f in (train, token):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = f()
        graphs.append((g, got))
    for turn in range(4):
        cu = _cu([[100, 60, 90], [250, 0, 0], [1, 2, 200], [80, 80, 80]][turn])
        seqs.cu_q.copy_(_i32(cu))
        cache.len_k.copy_(_i32([[3, 7], [125, 0], [1, 124], [64, 65]][turn]))
        q.copy_(_rand(gen, *q.shape, dtype=dtype))
        v.copy_(_rand(gen, *v.shape, dtype=dtype))
        want = train() + token()
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for a, b in zip(graphs[0][1] + graphs[1][1], want):
            assert torch.equal(a, b), turn
        exact = reference(q, k, v, **dict(ref, cu_q=cu))
        check("out", graphs[0][1][0], *exact["out"])


def test_only_the_gradients_that_are_asked_for():
    import imageni2r_amd as i2r
    gen = torch.Generator(DEV).manual_seed(3)
    q, k, v, table, seqs, _ = _make(gen, BF16, 64, 4, 2, [100, 60], bias=(16, 40, False), causal=True)
    dout = _rand(gen, *q.shape, dtype=BF16)
    all_ = _grads(q, k, v, table, seqs, dout)
    for name, at in (("dq", 0), ("dk", 1), ("dv", 2), ("dtable", 3)):
        ops = [q, k, v, table]
        ops[at] = ops[at].detach().requires_grad_(True)
        out = i2r.packed_attention(*ops[:3], seqs, bias=ops[3])
        assert torch.equal(torch.autograd.grad(out, ops[at], dout)[0], all_[name]), name
        with pytest.raises(RuntimeError):
            torch.autograd.grad(torch.autograd.grad(i2r.packed_attention(*ops[:3], seqs, bias=ops[3]).float().sum(),
                                                    ops[at], create_graph=True)[0].float().sum(), ops[at])


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("batch,longest", [(63, 9), (64, 9), (65, 130), (130, 40), (300, 5)])
def test_many_sequences(dtype, batch, longest):
    """More sequences than a wave has lanes, some of them empty."""
    gen = torch.Generator(DEV).manual_seed(batch)
    lens = torch.randint(0, longest + 1, (batch,), generator=gen, device=DEV).tolist()
    _all(gen, *_make(gen, dtype, 16, 2, 1, lens, bias=(8, 20, True), causal=batch % 2 == 0))


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,heads,kv", [(24, 40, 1), (64, 64, 1), (128, 48, 1), (32, 66, 2), (96, 7, 1), (128, 128, 64),
                                          (64, 96, 48)])
def test_wide_groups_and_many_key_heads(dtype, dim, heads, kv):
    """Groups of more heads than a tile has columns, tokens and prompts; enough key / value heads that none is split."""
    gen = torch.Generator(DEV).manual_seed(heads)
    _all(gen, *_make(gen, dtype, dim, heads, kv, [3, 90, 40], causal=True))
    _all(gen, *_make(gen, dtype, dim, heads, kv, [1, 2, 0, 1], [70, 300, 5, 1], bias=(16, 50, False), causal=True))


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("scale", [-0.7, 0.0, 0.3])
@pytest.mark.parametrize("lens_q,lens_k", [([40, 70], None), ([1, 3], [900, 1300])])
def test_scale(dtype, scale, lens_q, lens_k):
    gen = torch.Generator(DEV).manual_seed(4)
    _all(gen, *_make(gen, dtype, 40, 2, 2, lens_q, lens_k, causal=True), scale=scale)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,heads,kv", [(64, 4, 2), (128, 4, 4), (16, 6, 1)])
@pytest.mark.parametrize("room", [64, 2000])
def test_few_rows_with_gaps_and_hidden_values(dtype, dim, heads, kv, room):
    """A few tokens a sequence against short and long (split) keys: rows of no sequence around and behind them, and NaN and
    infinities in each sequence's last key, which only its last token sees."""
    import imageni2r_amd as i2r
    gen = torch.Generator(DEV).manual_seed(dim + room)
    cu_q, n, fill = [2, 5, 5, 8], 11, [room, 7, room - 3]
    q = _rand(gen, n, heads, dim, dtype=dtype)
    k, v = (_rand(gen, 3 * room + 5, kv, dim, dtype=dtype) for _ in range(2))
    cu_k = [room * b for b in range(4)]
    seqs = i2r.PackedSequences(_i32(cu_q), _i32(cu_k), len_k=_i32(fill), causal=True)
    dout = _rand(gen, n, heads, dim, dtype=dtype)
    want = reference(q, k, v, cu_q, cu_k, fill, True, dout=dout)
    last = [cu_k[b] + fill[b] - 1 for b in (0, 2)]
    k[last], v[last] = math.nan, math.inf
    ends, outside = [4, 7], [0, 1, 8, 9, 10]
    seen = torch.ones(n, dtype=torch.bool, device=DEV)
    seen[ends] = False
    out = i2r.packed_attention(q, k, v, seqs)
    check("out", out[seen], want["out"][0][seen], want["out"][1][seen])
    assert bool((out[outside] == 0).all()) and bool(torch.isnan(out[ends].float()).any(-1).all())
    mark = torch.full_like(q, 7.0)
    i2r.packed_attention(q, k, v, seqs, out=mark)
    assert bool((mark[outside] == 7).all()) and torch.equal(mark[[2, 3, 5, 6]], out[[2, 3, 5, 6]])
    got = _grads(q, k, v, None, seqs, dout)
    check("dq", got["dq"][seen], want["dq"][0][seen], want["dq"][1][seen])
    assert bool((got["dq"][outside] == 0).all())


@pytest.mark.parametrize("heads,kv", [(2, 2), (4, 1), (128, 64)])
@pytest.mark.parametrize("dim", [64, 128])
def test_fp16_gradients_beyond_the_lifted_range(heads, kv, dim):
    """p and ds carry 2^12 in fp16: gradients so large that a lifted ds leaves the type's range, and so small that an
    unlifted one would vanish."""
    gen = torch.Generator(DEV).manual_seed(dim)
    q, k, v, table, seqs, ref = _make(gen, F16, dim, heads, kv, [30, 65], bias=(8, 20, True))
    for size in (40.0, 2e-3):
        dout = _rand(gen, *q.shape, dtype=F16, size=size)
        want = reference(q, k, v, dout=dout, **ref)
        got = _grads(q, k, v, table, seqs, dout)
        for name, w in want.items():
            check(name, got[name], *w)


def test_out_of_its_own():
    import imageni2r_amd as i2r
    q, k, v, _, seqs, _ = _make(torch.Generator(DEV).manual_seed(1), BF16, 64, 2, 2, [40], fused=True)
    q = q.contiguous()
    with pytest.raises(ValueError, match="storage"):
        i2r.packed_attention(q, k, v, seqs, out=q)


def test_no_rows():
    import imageni2r_amd as i2r
    for dtype in (F32, BF16):
        q, k = torch.zeros(0, 2, 64, dtype=dtype, device=DEV), torch.ones(5, 2, 64, dtype=dtype, device=DEV)
        seqs = i2r.PackedSequences(_i32([0, 0]), _i32([0, 5]))
        assert i2r.packed_attention(q, k, k, seqs).shape == (0, 2, 64)
        got = _grads(q, k, k, None, seqs, q)
        assert bool((got["dk"] == 0).all()) and bool((got["dv"] == 0).all())
        seqs = i2r.PackedSequences(_i32([0, 5]), _i32([0, 0]))
        assert bool((i2r.packed_attention(k, q, q, seqs) == 0).all())
        got = _grads(k, q, q, None, seqs, k)
        assert bool((got["dq"] == 0).all()) and got["dk"].shape == (0, 2, 64)


def test_refusals():
    import imageni2r_amd as i2r
    gen = torch.Generator(DEV).manual_seed(3)
    q, k, v, table, seqs, _ = _make(gen, F32, 16, 4, 2, [10, 6], bias=(16, 40, False))
    at = i2r.packed_attention
    for bad, kind in ((dict(q=q.half()), TypeError), (dict(q=q.double(), k=k.double(), v=v.double()), TypeError),
                      (dict(q=q[:, :3]), ValueError), (dict(k=k[:-1], v=v[:-1]), ValueError), (dict(v=v[:, :1]), ValueError),
                      (dict(q=q[..., :12], k=k[..., :12], v=v[..., :12]), ValueError), (dict(k=k[..., :8]), ValueError),
                      (dict(q=q.cpu()), i2r.ops._lib.I2RError), (dict(q=q[0]), ValueError), (dict(q=None), TypeError),
                      (dict(seqs=None), TypeError), (dict(bias=table[:, :8]), ValueError), (dict(bias=table.half()), TypeError),
                      (dict(bias=table.cpu()), i2r.ops._lib.I2RError), (dict(bias=table.T.contiguous().T), ValueError),
                      (dict(out=q.half()), TypeError), (dict(out=q[:5]), ValueError),
                      (dict(seqs=i2r.PackedSequences(seqs.cu_q)), ValueError),
                      (dict(q=q.clone().requires_grad_(True), out=q.clone()), ValueError)):
        with pytest.raises(kind):
            at(**{**dict(q=q, k=k, v=v, seqs=seqs, bias=table), **bad})
    P = i2r.PackedSequences
    cu = seqs.cu_q
    for args, kw, kind in (((cu.long(),), {}, TypeError), ((cu[:1],), {}, ValueError), ((cu[::2],), {}, ValueError),
                           ((cu, cu[:2]), {}, ValueError), ((cu,), dict(len_k=cu), ValueError), ((None,), {}, TypeError),
                           ((cu,), dict(pos_q=cu), ValueError), ((cu, cu), dict(pos_q=cu, buckets=seqs.buckets), ValueError),
                           ((cu.cpu(),), {}, i2r.ops._lib.I2RError)):
        with pytest.raises(kind):
            P(*args, **kw)
    with pytest.raises(ValueError):  # positions of another number of rows
        at(q, k, v, P(cu, buckets=seqs.buckets, pos_q=cu), bias=table)


@pytest.mark.parametrize("rows", [1, 300])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_cache_that_holds_head_after_head(dtype, rows):
    """Heads 2^22 elements and more apart are read where they lie, in both directions and by the token kernel."""
    import imageni2r_amd as i2r
    from imageni2r_amd import packed
    gen = torch.Generator(DEV).manual_seed(41)
    room, dim, kv, heads, used = (1 << 15) + 8, 128, 2, 4, 700
    cache = torch.zeros(2, kv, room, dim, dtype=dtype, device=DEV)
    cache[:, :, :used] = _rand(gen, 2, kv, used, dim, dtype=dtype)
    k, v = cache[0].transpose(0, 1), cache[1].transpose(0, 1)
    assert k.stride(1) >= 1 << 22
    assert packed._rows(k, "k", dtype, k.device).data_ptr() == k.data_ptr()
    q, dout = _rand(gen, rows, heads, dim, dtype=dtype), _rand(gen, rows, heads, dim, dtype=dtype)
    seqs = i2r.PackedSequences(_i32([0, rows]), _i32([0, room]), len_k=_i32([used]), causal=True)
    got = _grads(q, k, v, None, seqs, dout)
    want = _grads(q, k.contiguous(), v.contiguous(), None, seqs, dout)
    for name in got:
        assert torch.equal(got[name], want[name]), name
    with torch.no_grad():
        assert torch.equal(i2r.packed_attention(q, k, v, seqs), i2r.packed_attention(q, k.contiguous(), v.contiguous(), seqs))


def test_observed_steps_of_series_without_steps():
    import imageni2r_amd as i2r
    seqs, order = i2r.PackedSequences.of_observed(torch.zeros(3, 0, dtype=torch.bool, device=DEV), i2r.RelativeBuckets())
    assert order.numel() == 0 and seqs.cu_q.tolist() == [0, 0, 0, 0] == seqs.cu_k.tolist()
    q = torch.zeros(0, 2, 8, device=DEV)
    assert i2r.packed_attention(q, q, q, seqs, bias=torch.zeros(2, 32, device=DEV)).shape == (0, 2, 8)
