"""What the attention of packed sequences and the learned relative position bias cost: cases, inputs, plain forms.

Two operators in four uses:

* ``attention``: softmax(scale * q k^T + bias) v over sequences of different lengths that lie one behind the other in
  one tensor, with or without a causal mask, with fewer key / value heads than query heads, and with a bias that is
  looked up in a learned table by the bucket of the distance between key and query;
* ``train``: the same with the gradients of q, k, v and the table;
* ``token``: the same for one (or a few) new tokens a sequence against a long cache;
* ``bias``: the bias alone as a dense (heads, queries, keys) tensor, with the table's gradient.

Where ``own`` is false `run` computes them from elementary torch operations on padded batches, in 32 bits.
"""
import math

import torch

own = False

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    none = dict(buckets=0, distance=0, two_sided=False, positions=False)
    return [
        # inference of a completion stage's encoder layer: the observed points of 32 weather series of 96 steps, 5 heads
        # of 8, every point sees every other one, biased by how far apart the two were measured
        dict(name="series_f32", op="attention", type="float32", heads=5, kv_heads=5, dim=8, batch=32, longest=96,
             causal=False, buckets=32, distance=128, two_sided=True, positions=True),
        # sixteen prompts of up to 1024 tokens with a one-sided bias, as a server packs them
        dict(name="prompts_bf16", op="attention", type="bfloat16", heads=16, kv_heads=4, dim=64, batch=16, longest=1024,
             causal=True, buckets=32, distance=128, two_sided=False, positions=False),
        # odd lengths and a head size between the tiles' sizes, both directions
        dict(name="odd_f16", op="attention", type="float16", heads=12, kv_heads=6, dim=80, batch=7, longest=1999,
             causal=False, **none),
        # one long document
        dict(name="document_bf16", op="attention", type="bfloat16", heads=16, kv_heads=2, dim=128, batch=1,
             longest=16384, causal=True, **none),
        # training that encoder layer on 32 series of up to 768 observed points
        dict(name="train_series_f32", op="train", type="float32", heads=5, kv_heads=5, dim=8, batch=32, longest=768,
             causal=False, buckets=32, distance=128, two_sided=True, positions=True),
        # a training batch of eight packed documents with a learned bias
        dict(name="train_packed_bf16", op="train", type="bfloat16", heads=16, kv_heads=4, dim=64, batch=8, longest=2048,
             causal=True, buckets=32, distance=128, two_sided=False, positions=False),
        # two long documents, grouped heads, no bias
        dict(name="train_long_bf16", op="train", type="bfloat16", heads=32, kv_heads=8, dim=128, batch=2, longest=4096,
             causal=True, **none),
        # the first token after a short prompt: latency
        dict(name="token_short_f16", op="token", type="float16", heads=8, kv_heads=8, dim=64, batch=1, longest=40,
             rows=1, causal=True, **none),
        # a serving step: one token for each of 64 users
        dict(name="token_batch_bf16", op="token", type="bfloat16", heads=32, kv_heads=8, dim=128, batch=64,
             longest=8192, rows=1, causal=True, **none),
        # one user with a very long cache and a bias
        dict(name="token_long_bf16", op="token", type="bfloat16", heads=32, kv_heads=8, dim=128, batch=1,
             longest=131072, rows=1, causal=True, buckets=32, distance=128, two_sided=False, positions=False),
        # a dense bias for a 96-step series' encoder, forward and gradient
        dict(name="bias_series_f32", op="bias", type="float32", heads=5, queries=96, keys=96, buckets=32, distance=128,
             two_sided=True, positions=True),
        # a dense bias over a long context
        dict(name="bias_long_bf16", op="bias", type="bfloat16", heads=16, queries=2048, keys=2048, buckets=32,
             distance=128, two_sided=True, positions=False),
    ]


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    while True:
        op = rng.choice(["attention", "attention", "train", "train", "token", "token", "bias"])
        kind = rng.choice(["float32", "bfloat16", "bfloat16", "float16"])
        case = dict(op=op, type=kind, buckets=0, distance=0, two_sided=False, positions=False)
        if op == "bias" or rng.random() < 0.5:
            case.update(buckets=2 * rng.randint(4, 32), distance=_log(rng, 64, 1024), two_sided=rng.random() < 0.5)
            case.update(positions=op != "token" and rng.random() < 0.5)
        if op == "bias":
            case.update(heads=_log(rng, 1, 32), queries=_log(rng, 1, 2500), keys=_log(rng, 1, 2500))
        else:
            kv = rng.choice([1, 2, 4, 5, 8])
            heads = kv * rng.choice([1, 1, 2, 3, 4, 8])
            case.update(heads=heads, kv_heads=kv, dim=8 * rng.randint(1, 16), batch=_log(rng, 1, 64),
                        # (the gradients of a lone token's weights are all zero)
                        longest=_log(rng, 4 if op == "train" else 1, 131072 if op == "token" else 8192),
                        causal=not case["two_sided"] and rng.random() < 0.7)
            if op == "token":
                case.update(rows=rng.choice([1, 1, 1, 2, 4]), causal=True)
                case["longest"] = max(case["longest"], case["rows"])
        if _cost(case) <= max(_cost(c) for c in listed() if c["op"] == op):
            return case


def _cost(case):
    """What a case costs the padded form, in elements of the widest tensors that it makes."""
    if case["op"] == "bias":
        return case["queries"] * case["keys"] * (2 * case["heads"] + case["buckets"])
    rows = case["rows"] if case["op"] == "token" else case["longest"]
    scores = case["batch"] * rows * case["longest"] * (case["heads"] + case["buckets"] * (case["op"] == "train"))
    wide = 4 if case["type"] == "float32" else 2
    return scores + case["batch"] * case["longest"] * case["kv_heads"] * case["dim"] * wide


def _lengths(case):
    """Lengths of the case's sequences: the longest first, the others spread down to 40 % of it."""
    n = case["longest"]
    return [max(1, n - int(0.6 * n * (i * 0.6180339887498949 % 1.0))) for i in range(case["batch"])]


def _bucket_of(case):
    """Bucket of every distance from 0 to `distance` in one direction, from whole numbers alone.

    Half of a direction's buckets hold one distance each; from there on bucket ``e + t`` begins at the first n with
    (n / e)^m >= (distance / e)^t, m the number of the other buckets, so that the last begins at or before `distance`.
    """
    half = case["buckets"] // 2 if case["two_sided"] else case["buckets"]
    e = half // 2
    m, far = half - e, case["distance"]
    return [n if n < e else min(half - 1, e + sum(n**m * e**t >= far**t * e**m for t in range(1, m)))
            for n in range(far + 1)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, device="cuda", generator=gen)  # noqa: E731
    whole = lambda values: torch.tensor(values, dtype=torch.int32, device="cuda")  # noqa: E731
    kind, heads = TYPES[case["type"]], case["heads"]
    state = dict(case=case)
    if case["buckets"]:
        state["table"] = normal(heads, case["buckets"])
        state["bucket_of"] = torch.tensor(_bucket_of(case), device="cuda")
    if case["op"] == "bias":
        if case["positions"]:  # the times at which points were observed, in order
            state["pos_q"] = (2 * case["queries"] * torch.rand(case["queries"], device="cuda", generator=gen)).int().sort().values
            state["pos_k"] = (2 * case["keys"] * torch.rand(case["keys"], device="cuda", generator=gen)).int().sort().values
        state["dout"] = normal(heads, case["queries"], case["keys"]).to(kind)
    else:
        lengths, dim, kv = _lengths(case), case["dim"], case["kv_heads"]
        starts = [sum(lengths[:i]) for i in range(len(lengths) + 1)]
        if case["op"] == "token":  # a cache with room for the longest sequence, and some new rows a sequence
            batch, rows, room = case["batch"], case["rows"], case["longest"] + 8
            state["cu_q"] = whole([rows * i for i in range(batch + 1)])
            state["cu_k"] = whole([room * i for i in range(batch + 1)])
            state["len_k"] = whole([max(n, rows) for n in lengths])
            state["q"] = normal(batch * rows, heads, dim).to(kind)
            state["k"] = normal(batch * room, kv, dim).to(kind)
            state["v"] = normal(batch * room, kv, dim).to(kind)
        else:  # one projection made q, k and v of each token side by side
            qkv = normal(starts[-1], heads + 2 * kv, dim).to(kind)
            state["cu_q"] = whole(starts)
            state["q"], state["k"], state["v"] = qkv[:, :heads], qkv[:, heads : heads + kv], qkv[:, heads + kv :]
            if case["positions"]:  # a sequence is the observed part of a series half as long again
                times = [torch.rand(n + n // 2, device="cuda", generator=gen).argsort()[:n].sort().values for n in lengths]
                state["pos_q"] = torch.cat(times).int()
        if case["op"] == "train":
            state["dout"] = normal(*state["q"].shape).to(kind)
            for name in ("q", "k", "v", "table"):
                if name in state:
                    state[name].requires_grad_(True)
    if own:
        import imageni2r_amd as i2r

        if case["buckets"]:
            state["buckets"] = i2r.RelativeBuckets(case["buckets"], case["distance"], bidirectional=case["two_sided"])
            if case["op"] == "bias":
                state["table"].requires_grad_(True)
        if case["op"] != "bias":
            state["seqs"] = i2r.PackedSequences(state["cu_q"], state.get("cu_k"), len_k=state.get("len_k"),
                                                causal=case["causal"], buckets=state.get("buckets"),
                                                pos_q=state.get("pos_q"))
    return state


def run(state):
    case = state["case"]
    if own:
        return _own(case, state)
    with torch.no_grad():
        return _plain_bias(case, state) if case["op"] == "bias" else _plain_attention(case, state)


def _own(case, s):
    import imageni2r_amd as i2r

    if case["op"] == "bias":
        out = i2r.relative_bias(s["table"], s["buckets"], case["queries"], case["keys"], pos_q=s.get("pos_q"),
                                pos_k=s.get("pos_k"), dtype=TYPES[case["type"]])
        return out.detach(), *torch.autograd.grad(out, s["table"], s["dout"])
    out = i2r.packed_attention(s["q"], s["k"], s["v"], s["seqs"], bias=s.get("table"))
    if case["op"] != "train":
        return out
    leaves = [s[name] for name in ("q", "k", "v", "table") if name in s]
    return out.detach(), *torch.autograd.grad(out, leaves, s["dout"])


# ------------------------------------------------------------------------------------------------ plain forms, 32 bits
def _plain_buckets(case, s, apart):
    """Bucket of each distance (key position less query position)."""
    half = case["buckets"] // 2
    if case["two_sided"]:
        return s["bucket_of"][apart.abs().clamp_max(case["distance"])] + half * (apart > 0)
    return s["bucket_of"][(-apart).clamp(0, case["distance"])]


def _plain_table_grad(case, bucket, grad):
    """Sums of grad (heads, rows, keys) over the places of each bucket, bucket (rows, keys)."""
    hot = (bucket[..., None] == torch.arange(case["buckets"], device="cuda")).float()
    return torch.matmul(grad.transpose(0, 1).contiguous(), hot).sum(0, dtype=torch.float64).float()


def _plain_bias(case, s):
    pos_q = s["pos_q"] if case["positions"] else torch.arange(case["queries"], device="cuda") + case["keys"] - case["queries"]
    pos_k = s["pos_k"] if case["positions"] else torch.arange(case["keys"], device="cuda")
    bucket = _plain_buckets(case, s, pos_k[None, :].long() - pos_q[:, None].long())
    return s["table"][:, bucket].to(TYPES[case["type"]]), _plain_table_grad(case, bucket, s["dout"].float())


def _plain_attention(case, s):
    heads, kv, dim, batch, kind = case["heads"], case["kv_heads"], case["dim"], case["batch"], TYPES[case["type"]]
    group, scale = heads // kv, case["dim"] ** -0.5
    cu_q = s["cu_q"].long()
    cu_k = s["cu_k"].long() if "cu_k" in s else cu_q
    len_q = cu_q[1:] - cu_q[:-1]
    len_k = s["len_k"].long() if "len_k" in s else cu_k[1:] - cu_k[:-1]
    n_q, n_k = case.get("rows", case["longest"]), max(case["longest"], case.get("rows", 1))
    iq, ik = torch.arange(n_q, device="cuda"), torch.arange(n_k, device="cuda")
    live_q, live_k = iq < len_q[:, None], ik < len_k[:, None]
    at_q = (cu_q[:-1, None] + iq).clamp_max(s["q"].shape[0] - 1)
    at_k = (cu_k[:-1, None] + ik).clamp_max(s["k"].shape[0] - 1)

    def rows_of(x, at, live):  # (n, h, d) -> (batch * kv, h / kv * rows, d), padded rows zero
        x = torch.where(live[..., None, None], x[at].float(), 0.0)
        return x.permute(0, 2, 1, 3).reshape(batch * kv, -1, dim)

    q, k, v = rows_of(s["q"], at_q, live_q), rows_of(s["k"], at_k, live_k), rows_of(s["v"], at_k, live_k)
    p = torch.matmul(q, k.transpose(1, 2).contiguous()).mul_(scale).view(batch, heads, n_q, n_k)
    seen = live_q[:, :, None] & live_k[:, None, :]
    if case["causal"]:
        seen &= ik <= iq[:, None] + (len_k - len_q)[:, None, None]
    if case["buckets"]:
        pos_q = s["pos_q"][at_q].long() if case["positions"] else iq + (len_k - len_q)[:, None]
        pos_k = s["pos_q"][at_k].long() if case["positions"] else ik.expand(batch, n_k)
        bucket = _plain_buckets(case, s, pos_k[:, None, :] - pos_q[:, :, None])
        p += s["table"][:, bucket].transpose(0, 1)
    p.masked_fill_(~seen[:, None], -math.inf)
    p.sub_(p.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)).exp_()
    p.div_(p.sum(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).tiny))
    flat = p.view(batch * kv, group * n_q, n_k)

    def packed(x, n, starts, count, total):  # (batch * kv, h / kv * n, d) -> (total, h, d), rows of no sequence zero
        x = x.view(batch, -1, n, dim).transpose(1, 2)
        row = torch.arange(total, device="cuda")
        b = (row[:, None] >= starts[None, 1:]).sum(1).clamp_max(batch - 1)
        i = row - starts[b]
        return torch.where((i < count[b])[:, None, None], x[b, i.clamp(0, n - 1)], 0.0).to(kind)

    out = packed(torch.matmul(flat, v), n_q, cu_q, len_q, s["q"].shape[0])
    if case["op"] != "train":
        return out
    do = rows_of(s["dout"], at_q, live_q)
    dv = torch.matmul(flat.transpose(1, 2), do)
    ds = torch.matmul(do, v.transpose(1, 2).contiguous())
    ds.sub_((ds * flat).sum(-1, keepdim=True)).mul_(flat)
    grads = [packed(torch.matmul(ds, k).mul_(scale), n_q, cu_q, len_q, s["q"].shape[0]),
             packed(torch.matmul(ds.transpose(1, 2), q).mul_(scale), n_k, cu_k, len_k, s["k"].shape[0]),
             packed(dv, n_k, cu_k, len_k, s["k"].shape[0])]
    if case["buckets"]:
        ds = ds.view(batch, heads, n_q, n_k).transpose(0, 1).reshape(heads, batch * n_q, n_k)
        grads.append(_plain_table_grad(case, bucket.view(batch * n_q, n_k), ds))
    return out, *grads


# --------------------------------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    s = {name: x.detach() if isinstance(x, torch.Tensor) else x for name, x in prepare(case, seed).items()}
    return _exact_bias(case, s) if case["op"] == "bias" else _exact_attention(case, s)


def _exact_slot(case, apart):
    """Bucket of each distance by the logarithms of the definition (a distance on a border belongs to the upper one)."""
    count = case["buckets"] // 2 if case["two_sided"] else case["buckets"]
    single = count // 2
    steps = apart.abs().double() if case["two_sided"] else torch.relu(-apart.double())
    along = torch.log(steps.clamp_min(1) / single) / math.log(case["distance"] / single)
    wide = (single + torch.floor((count - single) * along + 1e-9)).clamp_max(count - 1)
    slot = torch.where(steps < single, steps, wide)
    return (slot + count * (apart > 0) if case["two_sided"] else slot).long()


def _exact_bias(case, s):
    if case["positions"]:
        here, there = s["pos_q"].long(), s["pos_k"].long()
    else:
        here = torch.arange(case["keys"] - case["queries"], case["keys"], device="cuda")
        there = torch.arange(case["keys"], device="cuda")
    slot = _exact_slot(case, there - here[:, None])
    grad = s["dout"].double()
    sums = [torch.where(slot == i, grad, 0.0).sum((1, 2)) for i in range(case["buckets"])]
    return s["table"].double()[:, slot.reshape(-1)].reshape(grad.shape), torch.stack(sums, 1)


def _exact_attention(case, s):
    heads, per, train = case["heads"], case["heads"] // case["kv_heads"], case["op"] == "train"
    q, k, v = (s[x].double() for x in "qkv")
    out, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    dtable = torch.zeros(heads, max(1, case["buckets"]), dtype=torch.float64, device="cuda")
    begin_q, begin_k = s["cu_q"].tolist(), s.get("cu_k", s["cu_q"]).tolist()
    many_k = s["len_k"].tolist() if "len_k" in s else [b - a for a, b in zip(begin_k, begin_k[1:])]
    for b in range(case["batch"]):
        top, last = begin_q[b], begin_q[b + 1]
        low, n = begin_k[b], many_k[b]
        piece = max(1, (1 << 26) // max(n, 1))
        for first in range(top, last, piece):
            rows = slice(first, min(last, first + piece))
            order = torch.arange(rows.start - last, rows.stop - last, device="cuda") + n  # place among the keys
            behind = torch.arange(n, device="cuda")
            apart = behind - order[:, None]
            hidden = apart > 0
            if case["positions"]:
                apart = s["pos_q"][low : low + n].long() - s["pos_q"][rows].long()[:, None]
            slot = _exact_slot(case, apart) if case["buckets"] else None
            for h in range(heads):
                g = h // per
                score = (q[rows, h] @ k[low : low + n, g].T) / math.sqrt(case["dim"])
                if case["buckets"]:
                    score = score + s["table"][h].double()[slot]
                if case["causal"]:
                    score = torch.where(hidden, -math.inf, score)
                weight = torch.exp(score - torch.logsumexp(score, -1, keepdim=True))
                out[rows, h] = weight @ v[low : low + n, g]
                if train:
                    up = s["dout"][rows, h].double()
                    dv[low : low + n, g] += weight.T @ up
                    dscore = weight * (up @ v[low : low + n, g].T - (up * out[rows, h]).sum(-1, keepdim=True))
                    dq[rows, h] = dscore @ k[low : low + n, g] / math.sqrt(case["dim"])
                    dk[low : low + n, g] += dscore.T @ q[rows, h] / math.sqrt(case["dim"])
                    if case["buckets"]:
                        dtable[h] += torch.zeros_like(dtable[h]).index_add_(0, slot.reshape(-1), dscore.reshape(-1))
    if not train:
        return out
    return out, dq, dk, dv, *([dtable] if case["buckets"] else [])


# ------------------------------------------------------------------------------------------------------- what it costs
def work(case):
    wide = {"float32": 4, "bfloat16": 2, "float16": 2}[case["type"]]
    if case["op"] == "bias":  # the bias written, its gradient read; one addition each
        n = case["heads"] * case["queries"] * case["keys"]
        return {"bytes": 2 * n * wide + 8 * case["heads"] * case["buckets"], "flops": n}
    lengths, dim, heads, kv = _lengths(case), case["dim"], case["heads"], case["kv_heads"]
    if case["op"] == "token":
        rows, lengths = case["rows"] * len(lengths), [max(n, case["rows"]) for n in lengths]
        pairs = sum(case["rows"] * n - case["rows"] * (case["rows"] - 1) // 2 for n in lengths)
    else:
        rows = sum(lengths)
        pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lengths)
    table = 4 * heads * case["buckets"]
    once = wide * dim * (2 * rows * heads + 2 * sum(lengths) * kv) + table
    if case["op"] != "train":
        return {"bytes": once, "flops": 4 * dim * pairs * heads}
    # q, k, v and the output's gradient are read, the output and three gradients written; six products
    return {"bytes": 2 * once, "flops": 12 * dim * pairs * heads}
