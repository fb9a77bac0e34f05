"""Buckets, and what the packed-sequence operators refuse before anything is launched (no GPU needed)."""
import ctypes

import pytest
import torch

from tests.packed_reference import bucket_by_logarithms


@pytest.mark.parametrize("two_sided", [True, False])
@pytest.mark.parametrize("num", [4, 6, 10, 32, 50, 64])
@pytest.mark.parametrize("far", [33, 64, 100, 128, 777, 1024])
def test_buckets_against_the_logarithms(num, far, two_sided):
    from imageni2r_amd import RelativeBuckets
    apart = torch.arange(-1100, 1101)
    got = RelativeBuckets(num, far, two_sided).bucket(apart)
    assert torch.equal(got, bucket_by_logarithms(apart, num, far, two_sided))


def test_buckets_by_hand():
    from imageni2r_amd import RelativeBuckets
    b = RelativeBuckets(8, 16, False)  # e = 4: 0 1 2 3 | 4..5 | 6(5.66)..7 | 8..11 | from 12 (11.3) on
    assert b.bucket(-torch.arange(20)).tolist() == [0, 1, 2, 3, 4, 4, 5, 5, 6, 6, 6, 6] + [7] * 8
    assert b.bucket(torch.arange(4)).tolist() == [0] * 4
    both = RelativeBuckets(16, 16, True)
    assert both.bucket(torch.tensor([0, -1, 1, -16, 16, 999])).tolist() == [0, 1, 9, 7, 15, 15]


@pytest.mark.parametrize("args", [(7, 128, True), (2, 128, True), (1, 128, False), (66, 128, True), (32, 8, True),
                                  (32, 1025, True), (8, 4, False)])
def test_bucket_refusals(args):
    from imageni2r_amd import RelativeBuckets
    with pytest.raises(ValueError):
        RelativeBuckets(*args)


def test_no_cpu_fallback():
    import imageni2r_amd as i2r
    with pytest.raises(i2r.ops._lib.I2RError, match="no CPU fallback"):
        i2r.PackedSequences(torch.tensor([0, 4], dtype=torch.int32))
    with pytest.raises(i2r.ops._lib.I2RError, match="no CPU fallback"):
        i2r.relative_bias(torch.zeros(2, 8), i2r.RelativeBuckets(8, 20), 4, 4)


def _fwd(seqs=True, q=64, k=64, v=64, table=None, out=64, dtype=0, nq=4, nk=4, heads=2, kv=2, dim=16, strides=(32, 16) * 3,
         cu=64, lut=64, nb=8, far=20, pos=(None, None)):
    """The C entry with addresses that nothing reads: every refusal comes before a launch."""
    from imageni2r_amd import _lib, packed
    s = packed._Seqs(cu, cu, None, pos[0], pos[1], lut, 1, 0, nb, far)
    _lib.call("i2r_packed_attention_fwd", ctypes.byref(s) if seqs else None, q, k, v, table, out, None, None, None, 0, dtype,
              nq, nk, heads, kv, dim, *strides, 1.0, 1, None)


@pytest.mark.parametrize("bad", [dict(seqs=False), dict(cu=None), dict(dtype=3), dict(dtype=-1), dict(nq=-1), dict(heads=3),
                                 dict(heads=0), dict(kv=0), dict(dim=12), dict(dim=136), dict(dim=0), dict(q=None),
                                 dict(v=None), dict(q=72), dict(strides=(34, 16) * 3), dict(strides=(-32, 16) * 3),
                                 dict(pos=(64, None)), dict(table=64, lut=None), dict(table=64, nb=65), dict(table=64, nb=0),
                                 dict(table=64, far=1025), dict(out=None), dict(out=72)], ids=str)
def test_c_refusals_forward(bad):
    from imageni2r_amd import _lib
    with pytest.raises(_lib.I2RError):
        _fwd(**bad)


def test_c_refusals_backward():
    from imageni2r_amd import _lib, packed
    s = packed._Seqs(64, 64, None, None, None, 64, 1, 0, 8, 20)

    def call(out32=64, stats=64, dout=64, dq=64, dk=64, dv=64, table=64, dtable=64, ws=64, n=1 << 30, nb=8):
        s.num_buckets = nb
        _lib.call("i2r_packed_attention_bwd", ctypes.byref(s), 64, 64, 64, table, out32, stats, dout, dq, dk, dv, dtable, ws,
                  n, 0, 4, 4, 2, 2, 16, *(32, 16) * 3, 1.0, None)

    for bad in (dict(out32=None), dict(stats=None), dict(dout=None), dict(dk=None), dict(dv=None), dict(table=None),
                dict(ws=None), dict(n=8), dict(nb=65), dict(dout=72), dict(dq=72), dict(dk=72)):
        with pytest.raises(_lib.I2RError):
            call(**bad)


def test_c_refusals_bias():
    from imageni2r_amd import _lib
    for bad in (dict(table=None), dict(lut=None), dict(out=None), dict(dtype=3), dict(heads=0), dict(nq=-1), dict(nb=65),
                dict(far=-1), dict(pos_q=64)):
        a = {**dict(table=64, lut=64, pos_q=None, pos_k=None, out=64, dtype=0, heads=2, nq=4, nk=4, nb=8, far=20), **bad}
        with pytest.raises(_lib.I2RError):
            _lib.call("i2r_relative_bias_fwd", *a.values(), None)
        b = {**dict(dout=64, lut=64, pos_q=None, pos_k=None, dtable=64, ws=64, n=1 << 20, dtype=0, heads=2, nq=4, nk=4, nb=8,
                    far=20)}
        b.update({{"table": "dtable", "out": "dout"}.get(k, k): v for k, v in bad.items()})
        with pytest.raises(_lib.I2RError):
            _lib.call("i2r_relative_bias_bwd", *b.values(), None)
    with pytest.raises(_lib.I2RError):
        _lib.call("i2r_relative_bias_bwd", 64, 64, None, None, 64, 64, 0, 0, 2, 4, 4, 8, 20, None)


def test_sizes_of_workspaces_take_any_sizes():
    from imageni2r_amd import _lib
    assert _lib.query("i2r_relative_bias_bwd_ws_bytes", 0, 0, 0, 0) == 0
    for n in (0, 1, 7, 100000):
        assert _lib.query("i2r_packed_attention_fwd_ws_bytes", 2, 3, n, n, 8, 2, 64) >= 0
        assert _lib.query("i2r_packed_attention_bwd_ws_bytes", 2, 3, n, n, 8, 2, 64, 32) >= 0


def test_c_refuses_tokens_too_far_apart():
    from imageni2r_amd import _lib
    for i in (0, 2, 4):
        strides = [32, 16] * 3
        strides[i] = 1 << 22
        with pytest.raises(_lib.I2RError, match="below 2\\^22"):
            _fwd(strides=strides)
