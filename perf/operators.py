"""The dense attention operators that a hierarchical decoder needs next to its span attention, as measured cases.

Three ways in which a program meets them:

  forward  queries of one sequence over the states of another (an encoder's, of another length), for inference
  train    the same with its gradients for queries, keys and values
  decode   one new token of every sequence over a key/value cache that lives in pages

For every batch entry b and query head h (its key/value head is h // (heads / kv_heads)), with s = 1 / sqrt(head_dim):

  p[i, j] = exp(s q[i].k[j] - m[i]) / sum over attended j,     out[i] = sum over attended j of p[i, j] v[j]

A key is attended when its position is below the entry's length and the mask (if there is one) lets the query see it; a query
that sees no key gives zeros.  `run` computes this in elementary 32-bit operations, or calls the package where `own` is true.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# --------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # A short prompt over a short memory: the smallest call, where latency counts.
        _attention("forward prompt", "forward", "bf16", 1, 16, 77, 8, 8, 64),
        # A batch of decoder sequences over encoder states of ragged length, one of them absent.
        _attention("forward ragged memory", "forward", "bf16", 8, 2048, 1000, 8, 8, 64, lengths="ragged"),
        # The layer at its benchmark length: 16 heads of 128, 4096 rows on both sides.
        _attention("forward 4096 x 4096", "forward", "bf16", 4, 4096, 4096, 16, 16, 128),
        # A few new rows (a chunk of a prompt) over a long memory.
        _attention("forward few rows, long memory", "forward", "f16", 2, 33, 30011, 16, 16, 128),
        # Sequences packed into one row, each with its own stretch of the memory; padding rows see nothing.
        _attention("forward packed", "forward", "f16", 2, 1021, 1531, 8, 2, 96, mask="packed"),
        # Parity runs in 32 bits.
        _attention("train f32", "train", "f32", 2, 100, 130, 4, 4, 32, lengths="ragged"),
        # The training shape of the language model: 8 heads of 64, a memory shorter than the sequence.
        _attention("train ragged memory", "train", "bf16", 8, 2048, 515, 8, 8, 64, lengths="ragged"),
        # The layer at its benchmark length.
        _attention("train 4096 x 4096", "train", "bf16", 2, 4096, 4096, 16, 16, 128),
        # Shared key/value heads, odd lengths, some keys of each memory masked.
        _attention("train shared heads", "train", "f16", 3, 515, 1027, 12, 4, 128, mask="keys"),
        # One sequence, a short cache: latency.
        _decode("decode short", "bf16", 1, 8, 8, 64, 100, 16),
        # A batch of sequences of ragged length.
        _decode("decode batch", "bf16", 32, 16, 16, 128, 4096, 64, lengths="ragged"),
        # Few sequences, a long cache, query heads that share key/value heads.
        _decode("decode long", "f16", 2, 32, 4, 128, 131072, 256),
    ]


def _attention(name, kind, dtype, batch, queries, keys, heads, kv_heads, head_dim, lengths="full", mask="none"):
    return {"name": name, "kind": kind, "dtype": dtype, "batch": batch, "queries": queries, "keys": keys, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "lengths": lengths, "mask": mask}


def _decode(name, dtype, batch, heads, kv_heads, head_dim, keys, page, lengths="full"):
    return {"name": name, "kind": "decode", "dtype": dtype, "batch": batch, "queries": 1, "keys": keys, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "lengths": lengths, "mask": "none"}


def draw(rng):
    def span(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    while True:
        kind = rng.choice(["forward", "forward", "train", "train", "decode", "decode"])
        kv_heads = rng.choice([1, 2, 3, 4, 8, 12, 16])
        heads = kv_heads * rng.choice([1, 1, 1, 2, 4, 8])
        if heads > 32:
            continue
        if kind == "decode":
            case = _decode("", rng.choice(["bf16", "bf16", "f16", "f32"]), span(1, 64), heads, kv_heads,
                           rng.choice([32, 64, 64, 96, 128, 128]), span(1, 131072), rng.choice([16, 16, 32, 64, 128, 256]),
                           lengths=rng.choice(["full", "ragged"]))
            limit = 1.1e9
        else:
            dtype = rng.choice(["bf16", "bf16", "bf16", "f16", "f16", "f32"])
            case = _attention("", kind, dtype, span(1, 16), span(1, 4096), span(1, 32768), heads, kv_heads,
                              rng.choice([32, 64, 64, 96, 128, 128]), lengths=rng.choice(["full", "ragged"]),
                              mask=rng.choice(["none", "none", "none", "keys", "packed"]))
            limit = 2e9 if dtype == "f32" else 1e9                       # the 32-bit scores of the plain form, in elements
            if case["batch"] * heads * case["queries"] * case["keys"] > limit / 4 or (
                    dtype == "f32" and case["batch"] * heads * case["queries"] * case["keys"] > 2 ** 25):
                continue
            limit = 5e11
        w = work(case)
        if (w["bytes"] if kind == "decode" else w["flops"]) <= limit:
            del case["name"]
            return case


# -------------------------------------------------------------------------------------------------------------- inputs
def _lengths(case):
    """The multiset of lengths of a case (prepare() deals them out in an order of the seed's)."""
    batch, keys = case["batch"], case["keys"]
    if case["lengths"] == "full":
        return [keys] * batch
    got = [max(1, int(keys * ((0.618034 * i) % 1.0))) if i else keys for i in range(batch)]
    if batch >= 4:
        got[3] = 1
    if batch >= 6:
        got[5] = 0
    return got


def _segments(case):
    """Packed rows: (query rows, key rows) of every segment; the last rows of each side belong to none."""
    count = max(1, min(case["queries"], case["keys"], 5) - 1)
    q, k = int(case["queries"] * 0.95), int(case["keys"] * 0.97)
    if q < count or k < count:
        return []
    cut = lambda total: [total * (i + 1) * (i + 2) // (count * (count + 1)) for i in range(count)]      # noqa: E731
    qs, ks = cut(q), cut(k)
    return [(a - b, c - d) for a, b, c, d in zip(qs, [0] + qs, ks, [0] + ks)]


def _kept_keys(case):
    return max(1, int(case["keys"] * 0.8))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 2654435761 % (2 ** 31))
    dtype = _TYPES[case["dtype"]]
    batch, queries, keys = case["batch"], case["queries"], case["keys"]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["head_dim"]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32 if dtype == torch.float32 else dtype) * scale)

    order = torch.randperm(batch, generator=gen, device="cuda").tolist()
    sizes = [_lengths(case)[i] for i in order]
    state = {"case": case}
    if case["kind"] == "decode":
        page = case["page"]
        per_row = [-(-n // page) for n in sizes]
        width = max(1, max(per_row))
        pages = sum(per_row) + 1
        free = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
        table = torch.zeros(batch, width, dtype=torch.int32, device="cuda")
        at = 0
        for b, n in enumerate(per_row):
            table[b, :n] = free[at:at + n]
            at += n
        state["q"] = normal(batch, heads, dim, scale=1.5)
        state["k"] = normal(pages, page, kv_heads, dim)
        state["v"] = normal(pages, page, kv_heads, dim)
        state["table"] = table
        state["lengths"] = torch.tensor(sizes, dtype=torch.int32, device="cuda")
        return state
    state["q"] = normal(batch, queries, heads, dim, scale=1.5)
    state["k"] = normal(batch, keys, kv_heads, dim)
    state["v"] = normal(batch, keys, kv_heads, dim)
    if case["kind"] == "train":
        state["dout"] = normal(batch, queries, heads, dim)
    state["lengths"] = torch.tensor(sizes, dtype=torch.int32, device="cuda") if case["lengths"] != "full" else None
    state["mask"] = None
    if case["mask"] == "keys":
        rank = torch.rand(batch, keys, generator=gen, device="cuda").argsort(dim=1)
        mask = torch.zeros(batch, keys, dtype=torch.bool, device="cuda").scatter_(1, rank[:, :_kept_keys(case)], True)
        state["mask"] = mask.view(batch, 1, 1, keys)
    elif case["mask"] == "packed":
        mask = torch.zeros(batch, 1, queries, keys, dtype=torch.bool, device="cuda")
        parts = _segments(case)
        for b in range(batch):
            i = j = 0
            for s in torch.randperm(len(parts), generator=gen, device="cuda").tolist():
                mask[b, 0, i:i + parts[s][0], j:j + parts[s][1]] = True
                i, j = i + parts[s][0], j + parts[s][1]
        state["mask"] = mask
    return state


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    heads, kv_heads, dim, batch, queries, keys = (case[n] for n in ("heads", "kv_heads", "head_dim", "batch", "queries", "keys"))
    lengths = _lengths(case)
    pairs, seen = queries * sum(lengths), sum(lengths)
    mask_bytes = 0
    if case["mask"] == "keys":
        # the kept keys lie anywhere: a length keeps its share of them
        pairs, seen, mask_bytes = pairs * _kept_keys(case) // keys, seen * _kept_keys(case) // keys, batch * keys
    elif case["mask"] == "packed":
        share = sum(lengths) / (batch * keys)
        pairs = int(batch * sum(a * b for a, b in _segments(case)) * share)
        mask_bytes = batch * queries * keys
    q_bytes = batch * queries * heads * dim * size                  # queries, and the output of the same shape
    kv_bytes = 2 * seen * kv_heads * dim * size
    extra = mask_bytes + 4 * batch
    if case["kind"] == "train":
        # read q, k, v, dout; write out, dq, dk, dv (gradients of all rows); scores, weighted sum, and the four products of the backward
        return {"bytes": 4 * q_bytes + kv_bytes + 2 * batch * keys * kv_heads * dim * size + extra, "flops": 12 * pairs * heads * dim}
    if case["kind"] == "decode":
        extra += 4 * sum(-(-n // case["page"]) for n in lengths)
    return {"bytes": 2 * q_bytes + kv_bytes + extra, "flops": 4 * pairs * heads * dim}


# ----------------------------------------------------------------------------------------------------------- plain form
def _allowed(state, queries, keys):
    """[batch, 1 or heads, 1 or queries, keys] truth values, or None where every key is seen."""
    lengths, mask = state["lengths"], state.get("mask")
    allowed = None
    if lengths is not None:
        allowed = (torch.arange(keys, device="cuda") < lengths.view(-1, 1)).view(-1, 1, 1, keys)
    if mask is not None:
        allowed = mask if allowed is None else allowed & mask
    return allowed


def _weights(q, k, allowed, scale):
    """Softmax weights [B, Hkv, G, Lq, Lk] of q [B, Hkv, G, Lq, D] and k [B, Hkv, 1, Lk, D]; zeros where nothing is seen."""
    scores = torch.matmul(q * scale, k.transpose(-1, -2))
    if allowed is not None:
        allowed = allowed.unsqueeze(1)
        scores = torch.where(allowed, scores, -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    weights = torch.exp(scores.sub_(top))
    total = weights.sum(dim=-1, keepdim=True)
    return weights.div_(torch.where(total == 0.0, 1.0, total))


def _plain_attention(state):
    q, k, v = state["q"], state["k"], state["v"]
    batch, queries, heads, dim = q.shape
    keys, kv_heads = k.shape[1:3]
    group = heads // kv_heads
    scale = 1.0 / math.sqrt(dim)
    split = lambda t: t.float().view(batch, queries, kv_heads, group, dim).permute(0, 2, 3, 1, 4)            # noqa: E731
    join = lambda t: t.permute(0, 3, 1, 2, 4).reshape(batch, queries, heads, dim).to(q.dtype)              # noqa: E731
    per_key = lambda t: t.float().permute(0, 2, 1, 3).unsqueeze(2)                                         # noqa: E731
    qf, kf, vf = split(q), per_key(k), per_key(v)
    p = _weights(qf, kf, _allowed(state, queries, keys), scale)
    out = torch.matmul(p, vf)
    if "dout" not in state:
        return join(out)
    g = split(state["dout"])
    dv = torch.matmul(p.transpose(-1, -2), g).sum(dim=2)
    dp = torch.matmul(g, vf.transpose(-1, -2))
    ds = dp.sub_((g * out).sum(dim=-1, keepdim=True)).mul_(p).mul_(scale)
    dq = torch.matmul(ds, kf)
    dk = torch.matmul(ds.transpose(-1, -2), qf).sum(dim=2)
    back = lambda t: t.permute(0, 2, 1, 3).to(q.dtype)                                                     # noqa: E731
    return join(out), join(dq), back(dk).contiguous(), back(dv).contiguous()


def _plain_decode(state):
    q, table, lengths = state["q"], state["table"], state["lengths"]
    batch, heads, dim = q.shape
    page, kv_heads = state["k"].shape[1:3]
    keys = table.shape[1] * page
    group = heads // kv_heads
    k = state["k"][table.long()].view(batch, keys, kv_heads, dim).float().permute(0, 2, 1, 3).unsqueeze(2)
    v = state["v"][table.long()].view(batch, keys, kv_heads, dim).float().permute(0, 2, 1, 3).unsqueeze(2)
    qf = q.float().view(batch, kv_heads, group, 1, dim)
    allowed = (torch.arange(keys, device="cuda") < lengths.view(-1, 1)).view(batch, 1, 1, keys)
    p = _weights(qf, k, allowed, 1.0 / math.sqrt(dim))
    return torch.matmul(p, v).view(batch, heads, dim).to(q.dtype)


def run(state):
    kind = state["case"]["kind"]
    if own:
        from sparseattention_b200.ops import cross_attention, paged_attention_decode
        if kind == "decode":
            return paged_attention_decode(state["q"], state["k"], state["v"], state["table"], state["lengths"])
        q, k, v = state["q"], state["k"], state["v"]
        if kind == "forward":
            return cross_attention(q, k, v, key_lengths=state["lengths"], mask=state["mask"])
        q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
        out = cross_attention(q, k, v, key_lengths=state["lengths"], mask=state["mask"])
        return (out.detach(), *torch.autograd.grad(out, (q, k, v), state["dout"]))
    return _plain_decode(state) if kind == "decode" else _plain_attention(state)


# ---------------------------------------------------------------------------------------------------------- definition
def exact(case, seed):
    """The definition in 64 bits, one (batch entry, head) at a time, over the keys that are there and nothing else."""
    state = prepare(case, seed)
    q, k, v = state["q"], state["k"], state["v"]
    group = case["heads"] // case["kv_heads"]
    scale = case["head_dim"] ** -0.5
    decode = case["kind"] == "decode"
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    train = case["kind"] == "train"
    if train:
        dq, dk, dv = (torch.zeros(t.shape, dtype=torch.float64, device="cuda") for t in (q, k, v))
    for b in range(case["batch"]):
        n = case["keys"] if state["lengths"] is None else int(state["lengths"][b])
        if n == 0:
            continue
        if decode:
            rows = state["table"][b, : -(-n // case["page"])].long()
            kb, vb = (t[rows].flatten(0, 1)[:n] for t in (k, v))
        else:
            kb, vb = k[b, :n], v[b, :n]
        hidden = None
        if state.get("mask") is not None:
            hidden = ~state["mask"][b, 0, :, :n]
        for h in range(case["heads"]):
            kh, vh = kb[:, h // group].double(), vb[:, h // group].double()
            qh = (q[b, h].view(1, -1) if decode else q[b, :, h]).double()
            logits = (qh @ kh.T) * scale
            if hidden is not None:
                logits.masked_fill_(hidden, -math.inf)
            p = torch.softmax(logits, dim=1).nan_to_num_(nan=0.0)        # a row that sees nothing
            oh = p @ vh
            if decode:
                out[b, h] = oh.view(-1)
                continue
            out[b, :, h] = oh
            if train:
                g = state["dout"][b, :, h].double()
                dv[b, :n, h // group] += p.T @ g
                ds = p * (g @ vh.T - (g * oh).sum(1, keepdim=True)) * scale
                dq[b, :, h] = ds @ kh
                dk[b, :n, h // group] += ds.T @ qh
    return (out, dq, dk, dv) if train else out
