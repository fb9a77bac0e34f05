"""Attention over packed sequences and the learned relative position bias by buckets (csrc/packed_attention.hip,
csrc/relative_bias.hip).

Irregular series have another number of observed points each.  Instead of padding them, their rows lie one behind the
other in one tensor and `PackedSequences` says where each begins:

    buckets = RelativeBuckets(32, 128)                           # distances -> 32 buckets, both directions
    seqs = PackedSequences(cu, buckets=buckets, pos_q=times)     # one for all layers of a batch
    out = packed_attention(q, k, v, seqs, bias=table)            # (rows, heads, dim); differentiable in q, k, v, table

The same call serves a token against a cache: ``PackedSequences(cu_q, cu_k, len_k=filled, causal=True)``.  All index
arrays stay on the device and are read by the kernels, so a captured graph may be replayed with other lengths.
`relative_bias` makes the same bias as a dense tensor for an attention that takes an additive mask.

Neither exists in the reference, whose completion stage pads its series and masks keys.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd import forward_ad

from . import _lib, ops

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
MAX_BUCKETS, MAX_DISTANCE = 64, 1024


class _Seqs(ctypes.Structure):  # i2r_packed_seqs
    _fields_ = ([(n, ctypes.c_void_p) for n in ("cu_q", "cu_k", "len_k", "pos_q", "pos_k", "lut")]
                + [(n, ctypes.c_int) for n in ("batch", "causal", "num_buckets", "max_distance")])


def _index(t, name, numel=None, device=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a tensor, got {type(t)}")
    if t.dtype != torch.int32:
        raise TypeError(f"{name}: expected torch.int32, got {t.dtype}")
    if not t.is_cuda:
        raise _lib.I2RError(f"{name}: tensor is on {t.device}; the HIP path needs a 'cuda' (HIP) tensor and there is "
                            "no CPU fallback")
    if t.dim() != 1 or not t.is_contiguous():
        raise ValueError(f"{name}: expected a contiguous vector, got shape {tuple(t.shape)}")
    if numel is not None and t.numel() != numel:
        raise ValueError(f"{name}: expected {numel} entries, got {t.numel()}")
    if device is not None and t.device != device:
        raise ValueError(f"{name}: on {t.device}, the other tensors on {device}")
    return t


class RelativeBuckets:
    """Buckets of relative positions r = key position - query position.

    Of the m buckets of a direction (half of ``num_buckets`` when ``bidirectional``, else all) the first e = m // 2 hold
    one distance n each; the others widen with its logarithm up to ``max_distance``:
    e + floor((m - e) * ln(n / e) / ln(max_distance / e)), at most m - 1.  Keys behind the query (r > 0) take the upper
    half when ``bidirectional``; else they share bucket 0 with the distance 0."""

    def __init__(self, num_buckets=32, max_distance=128, bidirectional=True):
        num_buckets, max_distance = int(num_buckets), int(max_distance)
        m = num_buckets // 2 if bidirectional else num_buckets
        if bidirectional and num_buckets % 2:
            raise ValueError(f"RelativeBuckets: {num_buckets} buckets cannot be halved between two directions")
        if m < 2 or num_buckets > MAX_BUCKETS:
            raise ValueError(f"RelativeBuckets: {num_buckets} buckets: 2 a direction to {MAX_BUCKETS} are supported")
        if not m // 2 < max_distance <= MAX_DISTANCE:
            raise ValueError(f"RelativeBuckets: max_distance {max_distance} is not in {m // 2 + 1}..{MAX_DISTANCE}")
        self.num_buckets, self.max_distance, self.bidirectional = num_buckets, max_distance, bool(bidirectional)
        e = m // 2
        # bucket e + t begins at the first n with (n / e)^(m-e) >= (max_distance / e)^t, compared as whole numbers
        starts = [max_distance**t * e**(m - e) for t in range(1, m - e)]
        near, t = [], 0
        for n in range(max_distance + 1):
            while n >= e and t < len(starts) and n**(m - e) * e**(t + 1) >= starts[t]:
                t += 1
            near.append(n if n < e else e + t)
        behind = [m + b for b in near[1:]] if bidirectional else [0] * max_distance
        #: bucket of each distance from -max_distance to max_distance
        self.lut = torch.tensor(near[:0:-1] + [near[0]] + behind, dtype=torch.uint8)
        self._on = {}

    def bucket(self, apart):
        """Buckets of a tensor of relative positions (int64, on its device)."""
        at = apart.clamp(-self.max_distance, self.max_distance).long() + self.max_distance
        return self.lut.to(apart.device)[at].long()

    def on(self, device):
        """The device's copy of `lut`, made once."""
        lut = self._on.get(device)
        if lut is None:
            if torch.cuda.is_current_stream_capturing():
                raise _lib.I2RError("RelativeBuckets: first use on this device inside a stream capture; use them once before")
            lut = self._on[device] = self.lut.to(device)
        return lut


class PackedSequences:
    """Where each sequence of a packed batch lies, for all attention layers of a pass.

    ``cu_q`` (batch + 1): sequence b owns rows cu_q[b] .. cu_q[b+1] of q.  ``cu_k`` the same for k and v (None: as
    ``cu_q``), of which the first ``len_k[b]`` rows hold keys (None: all; a cache of fixed room is cu_k = room * b with
    len_k its fill).  ``causal``: of Lq queries and Lk keys query i sees the keys j <= i + Lk - Lq.  ``buckets`` for a
    learned bias: by ``pos_q`` / ``pos_k``, a position for each row of q and k (``pos_k`` None with ``cu_k`` None: as
    ``pos_q``), or without them by j and i + Lk - Lq.

    All arrays are int32 vectors on the HIP device, read by the kernels when they run: an object stays valid when their
    values change (a cache that grows, a replayed graph: ``seqs.len_k.copy_(...)``) -- between a forward and its backward
    they must not.  The attributes themselves are fixed: the kernels have the arrays' addresses from the start.  Nothing
    checks the values on the host: the kernels clamp them to the tensors they are used with, and sequences have to
    ascend."""

    def __init__(self, cu_q, cu_k=None, *, len_k=None, causal=False, buckets=None, pos_q=None, pos_k=None):
        _index(cu_q, "cu_q")
        dev, batch = cu_q.device, cu_q.numel() - 1
        if batch < 1:
            raise ValueError("cu_q: expected the starts of one sequence at least and the last one's end")
        if cu_k is None and pos_k is None:
            pos_k = pos_q
        if (pos_q is None) != (pos_k is None):
            raise ValueError("positions: pos_q and pos_k are given together")
        if pos_q is not None and buckets is None:
            raise ValueError("positions: only a relative position bias reads them, and buckets is None")
        self.cu_q = cu_q
        self.cu_k = cu_q if cu_k is None else _index(cu_k, "cu_k", batch + 1, dev)
        self.len_k = None if len_k is None else _index(len_k, "len_k", batch, dev)
        self.pos_q = None if pos_q is None else _index(pos_q, "pos_q", None, dev)
        self.pos_k = None if pos_k is None else _index(pos_k, "pos_k", None, dev)
        self.batch, self.causal, self.buckets, self.device = batch, bool(causal), buckets, dev
        self._lut = None if buckets is None else buckets.on(dev)
        ptr = [None if t is None else t.data_ptr()
               for t in (self.cu_q, self.cu_k, self.len_k, self.pos_q, self.pos_k, self._lut)]
        self._c = _Seqs(*ptr, batch, int(self.causal), buckets.num_buckets if buckets else 0,
                        buckets.max_distance if buckets else 0)
        self._ref = ctypes.byref(self._c)

    def __setattr__(self, name, value):
        if self.__dict__.get(name, value) is not value:  # (len_k += 1 sets the array that it wrote into)
            raise AttributeError(f"PackedSequences.{name} is fixed: write into the array (copy_), or make another object")
        super().__setattr__(name, value)

    def __delattr__(self, name):
        raise AttributeError(f"PackedSequences.{name} is fixed")

    @classmethod
    def from_lengths(cls, lengths, device="cuda", **kw):
        """Sequences of these lengths one behind the other (queries and keys alike)."""
        cu = [0]
        for n in lengths:
            cu.append(cu[-1] + int(n))
        return cls(torch.tensor(cu, dtype=torch.int32, device=device), **kw)

    @classmethod
    def of_observed(cls, mask, buckets=None):
        """For series whose every step asks but whose observed steps alone answer: ``mask`` (B, L) bool, True where a step
        was observed.  -> (sequences, order): queries are all B * L rows, keys the rows ``order`` of them, of which those
        of a series lie together (rows of ``order`` behind the last series' are no keys).  With ``buckets`` positions are
        the steps.  Nothing waits for the device."""
        if mask.dtype != torch.bool or mask.dim() != 2:
            raise TypeError(f"mask: expected a (B, L) bool tensor, got {tuple(mask.shape)} {mask.dtype}")
        B, L = mask.shape
        dev = mask.device
        cu_q = torch.arange(B + 1, dtype=torch.int32, device=dev) * L
        cu_k = torch.zeros(B + 1, dtype=torch.int32, device=dev)
        torch.cumsum(mask.sum(1, dtype=torch.int32), 0, out=cu_k[1:])
        order = (~mask).reshape(-1).to(torch.uint8).argsort(stable=True)
        pos = dict(pos_q=torch.arange(L, dtype=torch.int32, device=dev).repeat(B),
                   pos_k=(order % max(L, 1)).to(torch.int32)) if buckets is not None else {}
        return cls(cu_q, cu_k, buckets=buckets, **pos), order


def _rows(t, name, dtype, device):
    """A (rows, heads, dim) operand: in place where its rows are contiguous, 16-byte aligned and less than 2^22 elements
    apart (heads may lie any way apart), else a copy."""
    if t.dim() != 3:
        raise ValueError(f"{name}: expected (rows, heads, dim), got {tuple(t.shape)}")
    if t.dtype != dtype:
        raise TypeError(f"{name}: expected {dtype}, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name}: on {t.device}, the sequences on {device}")
    s0, s1, s2 = t.stride()
    whole = 4 if dtype is torch.float32 else 8
    if s2 != 1 or (s0 | s1) % whole or t.data_ptr() % 16 or s0 >= 1 << 22 or s1 >= 1 << 40:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _check(q, k, v, seqs, bias):
    if not isinstance(seqs, PackedSequences):
        raise TypeError(f"seqs: expected PackedSequences, got {type(seqs)}")
    for t, name in ((q, "q"), (k, "k"), (v, "v")):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name}: expected a tensor, got {type(t)}")
        if not t.is_cuda:
            raise _lib.I2RError(f"{name}: tensor is on {t.device}; the HIP path needs a 'cuda' (HIP) tensor and there "
                                "is no CPU fallback")
    dt = q.dtype
    if dt not in _DTYPES:
        raise TypeError(f"q: expected float32, float16 or bfloat16, got {dt}")
    dev = seqs.device
    q, k, v = _rows(q, "q", dt, dev), _rows(k, "k", dt, dev), _rows(v, "v", dt, dev)
    nq, heads, dim = q.shape
    nk, kv_heads, kdim = k.shape
    if k.shape != v.shape:
        raise ValueError(f"packed_attention: k {tuple(k.shape)} and v {tuple(v.shape)} differ")
    if kdim != dim or dim % 8 or not 8 <= dim <= 128:
        raise ValueError(f"packed_attention: head dims {dim} and {kdim}: alike, a multiple of 8 and at most 128")
    if kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise ValueError(f"packed_attention: {heads} query heads are no multiple of {kv_heads} key / value heads")
    if max(nq, nk) >= 1 << 30:
        raise ValueError("packed_attention: at most 2^30 - 1 rows")
    if seqs.cu_k is seqs.cu_q and nk != nq:
        raise ValueError(f"packed_attention: {nq} query rows but {nk} key rows under one cu_q")
    if seqs.pos_q is not None and (seqs.pos_q.numel() != nq or seqs.pos_k.numel() != nk):
        raise ValueError(f"packed_attention: positions of {seqs.pos_q.numel()} / {seqs.pos_k.numel()} rows for {nq} / "
                         f"{nk} rows of q / k")
    if bias is not None:
        if seqs.buckets is None:
            raise ValueError("packed_attention: a bias needs sequences with buckets")
        ops._chk(bias, "bias")
        if tuple(bias.shape) != (heads, seqs.buckets.num_buckets):
            raise ValueError(f"bias: expected ({heads}, {seqs.buckets.num_buckets}), got {tuple(bias.shape)}")
        if bias.device != dev:
            raise ValueError(f"bias: on {bias.device}, the sequences on {dev}")
    return q, k, v


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _call(device, name, *args):
    """The call on ``device``'s current stream, whichever device is current."""
    index = device.index
    if index == _current_device():
        _lib.call(name, *args, ops._stream() if _raw_stream is None else _raw_stream(index))
    else:
        with torch.cuda.device(device):
            _lib.call(name, *args, ops._stream())


_sizes = {}


def _workspace(device, name, *sizes):
    """-> (workspace or None, its address or None, its bytes) of an entry point for these sizes."""
    key = (name,) + sizes
    n = _sizes.get(key)
    if n is None:
        if len(_sizes) >= 4096:
            _sizes.clear()
        n = _sizes[key] = _lib.query(name, *sizes)
    if n <= 0:
        return None, None, 0
    ws = torch.empty((n,), dtype=torch.uint8, device=device)
    return ws, ws.data_ptr(), n


def packed_attention_fwd(q, k, v, seqs, bias=None, scale=None, out=None, save=False):
    """-> (out, out32, stats).  ``save``: out32 (out before its rounding; out itself in fp32) and stats are what
    `packed_attention_bwd` reads, else None."""
    q, k, v = _check(q, k, v, seqs, bias)
    nq, heads, dim = q.shape
    nk, kv_heads, _ = k.shape
    dt, dev = _DTYPES[q.dtype], seqs.device
    fresh = out is None
    if fresh:
        out = torch.empty((nq, heads, dim), dtype=q.dtype, device=dev)
    elif tuple(ops._chk(out, "out", q.dtype).shape) != (nq, heads, dim) or out.device != dev or out.data_ptr() % 16:
        raise ValueError(f"out: expected a 16-byte aligned ({nq}, {heads}, {dim}) tensor on {dev}")
    elif any(out.untyped_storage().data_ptr() == t.untyped_storage().data_ptr() for t in (q, k, v)) and out.numel():
        raise ValueError("out: shares its storage with q, k or v, which are read after the first rows are written")
    out32 = stats = None
    if save:
        out32 = out if dt == 0 else torch.empty((nq, heads, dim), dtype=torch.float32, device=dev)
        stats = torch.empty((2, heads, nq), dtype=torch.float32, device=dev)
    ws, at, n = _workspace(dev, "i2r_packed_attention_fwd_ws_bytes", dt, seqs.batch, nq, nk, heads, kv_heads, dim)
    _call(dev, "i2r_packed_attention_fwd", seqs._ref, q.data_ptr(), k.data_ptr(), v.data_ptr(),
          None if bias is None else bias.data_ptr(), out.data_ptr(), None if dt == 0 or not save else out32.data_ptr(),
          None if stats is None else stats.data_ptr(), at, n, dt, nq, nk, heads,
          kv_heads, dim, q.stride(0), q.stride(1), k.stride(0), k.stride(1), v.stride(0), v.stride(1),
          float(dim**-0.5 if scale is None else scale), int(fresh))
    return out, out32, stats


def packed_attention_bwd(q, k, v, seqs, bias, out32, stats, dout, scale=None, need_dq=True, need_dkv=True,
                         need_dbias=True):
    """-> (dq, dk, dv, dbias), each None where it is not needed."""
    q, k, v = _check(q, k, v, seqs, bias)
    nq, heads, dim = q.shape
    nk, kv_heads, _ = k.shape
    dt, dev = _DTYPES[q.dtype], seqs.device
    dout = ops._chk(dout, "dout", q.dtype)
    if dout.data_ptr() % 16:
        dout = dout.clone()
    ops._chk(out32, "out32")
    ops._chk(stats, "stats")
    if dout.shape != q.shape or out32.shape != q.shape or tuple(stats.shape) != (2, heads, nq):
        raise ValueError("packed_attention_bwd: dout, out32 or stats have the wrong shape")
    if dout.device != dev or out32.device != dev or stats.device != dev:
        raise ValueError(f"packed_attention_bwd: dout, out32 or stats are not on {dev}")
    need_dbias = need_dbias and bias is not None
    nb = seqs.buckets.num_buckets if need_dbias else 0
    dq = torch.empty((nq, heads, dim), dtype=q.dtype, device=dev) if need_dq else None
    dk = torch.empty((nk, kv_heads, dim), dtype=q.dtype, device=dev) if need_dkv else None
    dv = torch.empty_like(dk) if need_dkv else None
    dbias = torch.empty((heads, nb), dtype=torch.float32, device=dev) if need_dbias else None
    ws, at, n = _workspace(dev, "i2r_packed_attention_bwd_ws_bytes", dt, seqs.batch, nq, nk, heads, kv_heads, dim, nb)
    _call(dev, "i2r_packed_attention_bwd", seqs._ref, q.data_ptr(), k.data_ptr(), v.data_ptr(),
          None if bias is None else bias.data_ptr(), out32.data_ptr(), stats.data_ptr(), dout.data_ptr(),
          *(None if t is None else t.data_ptr() for t in (dq, dk, dv, dbias)), at, n, dt, nq, nk, heads, kv_heads, dim,
          q.stride(0), q.stride(1), k.stride(0), k.stride(1), v.stride(0), v.stride(1),
          float(dim**-0.5 if scale is None else scale))
    return dq, dk, dv, dbias


def _differentiated(*tensors):
    """Whether autograd has to see the call: an input that asks for a gradient, or one that carries a tangent -- which the
    functions below have no derivative for, so that torch refuses it."""
    dual = getattr(forward_ad, "_current_level", 0) >= 0  # without an open dual level there are no tangents
    if dual or torch.is_grad_enabled():
        for t in tensors:
            if isinstance(t, torch.Tensor) and (t.requires_grad and torch.is_grad_enabled() or
                                                dual and forward_ad.unpack_dual(t).tangent is not None):
                return True
    return False


class PackedAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, bias, seqs, scale):
        out, out32, stats = packed_attention_fwd(q, k, v, seqs, bias, scale, save=True)
        ctx.save_for_backward(q, k, v, bias, out32, stats)
        ctx.seqs, ctx.scale = seqs, scale
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, bias, out32, stats = ctx.saved_tensors
        nq, nk, nv, nb = ctx.needs_input_grad[:4]
        dq, dk, dv, dbias = packed_attention_bwd(q, k, v, ctx.seqs, bias, out32, stats, ops._c(dout), ctx.scale,
                                                 need_dq=nq, need_dkv=nk or nv, need_dbias=nb)
        return dq, dk if nk else None, dv if nv else None, dbias, None, None


def packed_attention(q, k, v, seqs, bias=None, scale=None, out=None):
    """softmax(scale * q k^T + bias) v within each sequence of ``seqs`` -> (rows of q, heads, dim).

    q (rows, heads, dim); k, v (rows, kv_heads, dim), query head h reading key / value head h // (heads // kv_heads);
    float32, float16 or bfloat16, dim a multiple of 8 up to 128.  Views (one projection's output split into q, k, v; a
    cache, token by token or head by head) are read in place where their rows are contiguous, 16-byte aligned and less than
    2^22 elements apart, others are copied.  ``bias``: fp32
    (heads, num_buckets) table of the sequences' buckets.  ``scale``: dim ** -0.5 by default.  A query without keys gets
    0; a key of score -inf counts as hidden.  Rows of q in no sequence come out 0 -- with ``out`` (inference only, storage
    of its own) they are left as they were.  Differentiable in q, k, v and bias, backward and once (tangents are refused); the
    gradients' sums have a fixed order.

    Where a sequence has few queries (their mean number times the query heads that share a key / value head is at most
    32) the keys are split over workgroups, as a token against its cache wants it: batches that mix prompts and single
    tokens are faster in two calls.  In fp16 a score's gradient of 16 and more (from an output gradient that was scaled
    up) takes its rows off the matrix cores, at 50 times the time and more; bf16 has no such limit.

    A stream capture of forward and backward calls packed_attention_fwd and packed_attention_bwd, or captures the whole
    training step; autograd's own graph of an earlier eager pass must not be alive then (torch ends the process)."""
    if _differentiated(q, k, v, bias):
        if out is not None:
            raise ValueError("packed_attention: out= cannot be differentiated")
        return PackedAttentionFn.apply(q, k, v, bias, seqs, scale)
    return packed_attention_fwd(q, k, v, seqs, bias, scale, out)[0]


def _check_bias(table, buckets, q_len, k_len, pos_q, pos_k, dtype):
    if not isinstance(buckets, RelativeBuckets):
        raise TypeError(f"buckets: expected RelativeBuckets, got {type(buckets)}")
    ops._chk(table, "table")
    if table.dim() != 2 or table.shape[0] < 1 or table.shape[1] != buckets.num_buckets:
        raise ValueError(f"table: expected (heads, {buckets.num_buckets}), got {tuple(table.shape)}")
    if not 0 <= q_len < 1 << 30 or not 0 <= k_len < 1 << 30:
        raise ValueError(f"relative_bias: bad lengths {q_len}, {k_len}")
    if (pos_q is None) != (pos_k is None):
        raise ValueError("positions: pos_q and pos_k are given together")
    if pos_q is not None:
        _index(pos_q, "pos_q", q_len, table.device)
        _index(pos_k, "pos_k", k_len, table.device)
    if dtype not in _DTYPES:
        raise TypeError(f"relative_bias: expected float32, float16 or bfloat16, got {dtype}")


def relative_bias_fwd(table, buckets, q_len, k_len, pos_q=None, pos_k=None, dtype=torch.float32):
    _check_bias(table, buckets, q_len, k_len, pos_q, pos_k, dtype)
    out = torch.empty((table.shape[0], q_len, k_len), dtype=dtype, device=table.device)
    _call(table.device, "i2r_relative_bias_fwd", table.data_ptr(), buckets.on(table.device).data_ptr(), ops._p(pos_q),
          ops._p(pos_k), out.data_ptr(), _DTYPES[dtype], table.shape[0], q_len, k_len, buckets.num_buckets,
          buckets.max_distance)
    return out


def relative_bias_bwd(dout, buckets, pos_q=None, pos_k=None):
    """-> the table's gradient (heads, num_buckets) fp32."""
    if dout.dtype not in _DTYPES:
        raise TypeError(f"dout: expected float32, float16 or bfloat16, got {dout.dtype}")
    ops._chk(dout, "dout", dout.dtype)
    heads, q_len, k_len = dout.shape
    dtable = torch.empty((heads, buckets.num_buckets), dtype=torch.float32, device=dout.device)
    _check_bias(dtable, buckets, q_len, k_len, pos_q, pos_k, dout.dtype)
    ws, at, n = _workspace(dout.device, "i2r_relative_bias_bwd_ws_bytes", heads, q_len, k_len, buckets.num_buckets)
    _call(dout.device, "i2r_relative_bias_bwd", dout.data_ptr(), buckets.on(dout.device).data_ptr(), ops._p(pos_q),
          ops._p(pos_k), dtable.data_ptr(), at, n, _DTYPES[dout.dtype], heads, q_len, k_len, buckets.num_buckets,
          buckets.max_distance)
    return dtable


class RelativeBiasFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, buckets, q_len, k_len, pos_q, pos_k, dtype):
        ctx.cfg = (buckets, pos_q, pos_k)
        return relative_bias_fwd(table, buckets, q_len, k_len, pos_q, pos_k, dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        buckets, pos_q, pos_k = ctx.cfg
        return (relative_bias_bwd(ops._c(dout), buckets, pos_q, pos_k),) + (None,) * 6


def relative_bias(table, buckets, q_len, k_len, pos_q=None, pos_k=None, dtype=torch.float32):
    """The bias of ``table`` (heads, num_buckets) fp32 as a dense (heads, q_len, k_len) tensor of ``dtype``, for an
    attention that takes an additive mask.  Positions: int32 vectors, or None: key j at j, query i at i + k_len - q_len.
    Differentiable in ``table``, backward and once; the gradient's sums have a fixed order."""
    if _differentiated(table):
        return RelativeBiasFn.apply(table, buckets, q_len, k_len, pos_q, pos_k, dtype)
    return relative_bias_fwd(table, buckets, q_len, k_len, pos_q, pos_k, dtype)
