"""Dense attention: what single entries of K, of weights and of output gradients do to a result, kernel by kernel (algo 2: tensor
cores, 1: 32 bits).

With u = eps / 2 of the type of the tensors (half a step) and w = 2^-24 as in the other tests of this operator.
"""
import math

import pytest
import torch

from sparseattention_b200.ops import cross_attention, paged_attention_decode
from sparseattention_b200.ops.dense import dense_attention_backward, dense_attention_forward
from tests.test_dense_gpu import SHAPES, check, make

pytestmark = pytest.mark.gpu



def normal(*shape, dtype, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=gen, device="cuda").to(dtype)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("algo", [1, 2])
def test_one_nan_key_shows_wherever_it_lies(D, dtype, algo):
    """Every place of a tile that is computed in a way of its own: pairs of keys in turn, both members, both halves, and the tail."""
    q, k, v = (normal(1, n, 1, D, dtype=dtype, seed=n) for n in (130, 300, 300))
    for key in (*range(8), *range(64, 72), 127, 128, 131, 255, 256, 299):
        bad = k.clone()
        bad[0, key] = math.nan
        out, _, lse = dense_attention_forward(q, bad, v, scale=D ** -0.5, algo=algo)
        assert out.isnan().all() and lse.isnan().all(), key


@pytest.mark.parametrize("algo", [1, 2])
def test_infinite_scores(algo):
    """Finite bfloat16 rows whose product passes the largest 32-bit number.  An infinite score makes its row NaN, as inf - inf does
    in the definition; minus infinity is a weight of zero."""
    q, k, v = (normal(1, n, 1, 64, dtype=torch.bfloat16, seed=n) for n in (130, 300, 300))
    q[..., 0], k[..., 0] = 0.0, 0.0
    q[0, 17, 0, 0] = 3e38
    for key in (*range(8), 65, 70, 130, 298):
        for sign in (1.0, -1.0):
            one = k.clone()
            one[0, key, 0, 0] = sign * 3e38
            out, _, lse = dense_attention_forward(q, one, v, scale=0.125, algo=algo)
            s = 0.125 * q[0, :, 0].double() @ k[0, :, 0].double().T
            if sign < 0:
                s[17, key] = -math.inf
            want = torch.softmax(s, -1) @ v[0, :, 0].double()
            rest = torch.arange(130, device="cuda") != 17 if sign > 0 else slice(None)
            # weights and result rounded once each, and the rest of the arithmetic (a dot product of 64, exponentials) below 2^-15
            near = torch.softmax(s, -1) @ v[0, :, 0].double().abs() * (2.0 ** -8 + 2.0 ** -15) + want.abs() * 2.0 ** -8
            assert ((out[0, :, 0].double() - want).abs() <= near)[rest].all(), (key, sign)
            assert lse[0, rest, 0].isfinite().all()
            if sign > 0:
                assert out[0, 17].isnan().all() and not lse[0, 17].isfinite().any(), key


def definition(q, k, v, g, allowed=None):
    """(out, dq, dk, dv, ds) in 64 bits; allowed [B, H or 1, Lq or 1, Lk]."""
    B, Lq, H, D = q.shape
    Lk, Hkv = k.shape[1:3]
    heads = lambda t: t.double().permute(0, 2, 1, 3).repeat_interleave(H // t.size(2), dim=1)                # noqa: E731
    qd, kd, vd, gd = (heads(t) for t in (q, k, v, g))
    s = D ** -0.5 * qd @ kd.transpose(-1, -2)
    if allowed is not None:
        s = s.masked_fill(~allowed, -math.inf)
        vd = torch.where(allowed.expand(B, H, Lq, Lk).any(2).unsqueeze(-1), vd, 0.0)
    p = torch.softmax(s, -1).nan_to_num(nan=0.0)
    out = p @ vd
    ds = p * (gd @ vd.transpose(-1, -2) - (gd * out).sum(-1, keepdim=True))
    group = lambda t: t.view(B, Hkv, H // Hkv, Lk, D).sum(2).permute(0, 2, 1, 3)                             # noqa: E731
    back = lambda t: t.permute(0, 2, 1, 3)                                                                   # noqa: E731
    return (back(out), back(D ** -0.5 * ds @ kd), group(D ** -0.5 * ds.transpose(-1, -2) @ qd), group(p.transpose(-1, -2) @ gd), ds)


def run_training(q, k, v, g, algo=2, **kw):
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    return torch.autograd.grad(cross_attention(*leaves, algo=algo, **kw), leaves, g)


def as_good_as_rounded(got, want, what):
    """Off in norm by no more than rounding the exact result costs, plus twice half a step: weights and score gradients are rounded
    once each, relative to their own size, and errors of independent signs add up as the terms themselves do."""
    u = 2.0 ** -11
    floor = float((want.half().double() - want).norm() / want.norm())
    err = float((got.double() - want).norm() / want.norm())
    assert err <= floor + 2 * u, f"{what}: {err:.3g}, the result's own rounding {floor:.3g}"


@pytest.mark.parametrize("case", [(1, 64, 8192, 2, 1, 64, 1e-3), (1, 64, 32768, 2, 2, 64, 1e-2), (1, 64, 32768, 1, 1, 64, 1e-3),
                                  (2, 200, 5000, 4, 2, 128, 1e-3), (1, 6000, 40, 2, 1, 64, 1e-4), (2, 300, 2000, 2, 2, 72, 1e-3)])
def test_float16_gradients_of_long_rows(case):
    """Weights of about 1 / Lk and small output gradients: as float16 their score gradients are below 2^-14, or below 2^-24."""
    *(B, Lq, Lk, H, Hkv, D), size = case
    q, k, v = (normal(B, n, h, D, dtype=torch.float16, seed=n + h) for n, h in ((Lq, H), (Lk, Hkv), (Lk + 1, Hkv)))
    v = v[:, :Lk].contiguous()
    g = (normal(B, Lq, H, D, dtype=torch.float32, seed=5) * size).half()
    _, *want, _ = definition(q, k, v, g)
    for name, a, b in zip(("dq", "dk", "dv"), run_training(q, k, v, g), want):
        as_good_as_rounded(a, b, name)


def test_float16_score_gradients_beyond_the_type():
    q, k, v, g = (normal(2, n, 2, 64, dtype=torch.float32, seed=i) for i, n in enumerate((8, 3, 3, 8)))
    q, k, v, g = (q * 0.05).half(), (k * 0.05).half(), (v * 3).half(), (g * 12000).half()
    _, *want, ds = definition(q, k, v, g)
    assert float(ds.abs().max()) > 65504 and all(float(t.abs().max()) < 65504 for t in want)
    for name, a, b in zip(("dq", "dk", "dv"), run_training(q, k, v, g), want):
        as_good_as_rounded(a, b, name)


def test_float16_gradients_of_unequal_size():
    """Rows, heads and batch entries whose output gradients differ by powers of ten, and none at all."""
    B, Lq, Lk, H, Hkv, D = 3, 150, 3000, 4, 2, 64
    q, k, v = (normal(B, n, h, D, dtype=torch.float16, seed=n) for n, h in ((Lq, H), (Lk, Hkv), (Lk, Hkv)))
    g = normal(B, Lq, H, D, dtype=torch.float32, seed=6)
    g[0] *= 1e-3
    g[1, :, 2:] *= 1e-2
    g[1, ::2] *= 0.05
    g[2] = 0
    g = g.half()
    dq, dk, dv = run_training(q, k, v, g)
    _, wq, wk, wv, _ = definition(q, k, v, g)
    assert not dq[2].any() and not dk[2].any() and not dv[2].any()
    as_good_as_rounded(dq[0], wq[0], "dq of small gradients")
    for part in (slice(0, None, 2), slice(1, None, 2)):
        for heads in (slice(0, 2), slice(2, 4)):
            as_good_as_rounded(dq[1, part, heads], wq[1, part, heads], "dq of some rows")
    for name, a, b in (("dk", dk, wk), ("dv", dv, wv)):
        for at in ((0, slice(None), 0), (0, slice(None), 1), (1, slice(None), 0), (1, slice(None), 1)):
            as_good_as_rounded(a[at], b[at], name)


@pytest.mark.parametrize("D", [64, 72, 128])
@pytest.mark.parametrize("kind", ["lengths", "keys", "heads"])
def test_float16_hidden_rows_have_no_say(D, kind):
    """What lies in rows of V that nobody looks at (NaN, infinities, the largest numbers) changes no bit of a gradient."""
    B, Lq, Lk, H, Hkv = 2, 140, 700, 4, 2
    q, k, v, g = (normal(B, n, h, D, dtype=torch.float16, seed=n + h) for n, h in ((Lq, H), (Lk, Hkv), (Lk + 2, Hkv), (Lq + 1, H)))
    v, g = v[:, :Lk].contiguous(), g[:, :Lq].contiguous()
    kw = {}
    if kind == "lengths":
        kw["key_lengths"] = torch.tensor([531, 0], dtype=torch.int32, device="cuda")
        hidden = torch.arange(Lk, device="cuda") >= kw["key_lengths"].view(-1, 1)
        hidden = hidden.view(B, Lk, 1).expand(B, Lk, Hkv)
        allowed = ~hidden[..., 0].view(B, 1, 1, Lk)
    else:
        mask = torch.rand(B, H if kind == "heads" else 1, 1, Lk, device="cuda") < 0.4
        kw["mask"] = allowed = mask
        hidden = ~mask.expand(B, H, 1, Lk).view(B, Hkv, H // Hkv, Lk).any(2).transpose(1, 2)
    want = run_training(q, k, v, g, **kw)
    for value in (math.nan, math.inf, 65504.0):
        bad = v.clone()
        bad[hidden] = value
        assert all(torch.equal(a, b) for a, b in zip(run_training(q, k, bad, g, **kw), want))
    if kind != "lengths":
        _, *exact, _ = definition(q, k, v, g, allowed)
        for name, a, b in zip(("dq", "dk", "dv"), want, exact):
            as_good_as_rounded(a, b, name)


@pytest.mark.parametrize("shape", [s for s in SHAPES if s[5] % 8 == 0 and s[5] <= 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_tensor_core_kernels_by_name(shape, dtype):
    check(*make(*shape, dtype, seed=sum(shape)), algo=2)


# one key, few, a tail, whole tiles, and few rows over many keys (ranges that are joined)
RESTS = [(1, 5, 1, 2, 1, 64), (2, 40, 3, 2, 2, 64), (2, 130, 300, 4, 2, 128), (1, 300, 513, 2, 2, 72), (1, 40, 6000, 2, 1, 64),
         (1, 3, 20000, 2, 2, 128)]


@pytest.mark.parametrize("shape", RESTS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("algo", [1, 2])
def test_what_rounding_took_is_kept(shape, dtype, algo):
    """Queries of zeros weigh all keys alike, in numbers that every kernel holds exactly: output and rest together are the mean of the
    values up to the 32-bit sum (2 sqrt(n) + 8 half steps w of the magnitudes, 2^-21 for the exponentials of zero and the division)
    and the rest's own rounding, u of u |out|, or half of float16's smallest step."""
    B, Lq, Lk, H, Hkv, D = shape
    u, w, tiny = torch.finfo(dtype).eps / 2, 2.0 ** -24, 2.0 ** -25 if dtype == torch.float16 else 0.0
    q, _, v, _ = make(*shape, dtype, seed=Lk)
    k = make(*shape, dtype, seed=Lk + 1)[1]
    lengths = torch.tensor([Lk, Lk // 2][:B], dtype=torch.int32, device="cuda")
    out, rest, lse = dense_attention_forward(torch.zeros_like(q), k, v, lengths, scale=0.125, algo=algo)
    for b, n in enumerate(lengths.tolist()):
        vd = v[b, :n].double().repeat_interleave(H // Hkv, dim=1)                                            # [n, H, D]
        want, size = vd.mean(0), vd.abs().mean(0)
        total = out[b].double() + rest[b].double()
        tol = u * u * want.abs() + ((2 * math.sqrt(n) + 8) * w + 2.0 ** -21) * size + tiny
        assert ((total - want).abs() <= tol).all()
        assert (rest[b].double().abs() <= u * out[b].double().abs() * (1 + 2 * u) + tiny).all()
        assert ((lse[b].double() - math.log(n)).abs() <= (math.log(n) + 4) * 2.0 ** -22).all()


@pytest.mark.parametrize("keys", [2, 3])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("algo", [1, 2])
def test_the_rest_carries_gradients_over_few_keys(keys, dtype, algo):
    """Values that differ by a step or two of their type, under equal weights: the gradients of the scores are differences of numbers
    that agree in their leading bits, and the output's rounding alone is as large as they are."""
    B, Lq, H, D, scale = 2, 70, 2, 64, 0.125
    u, w = torch.finfo(dtype).eps / 2, 2.0 ** -24
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    q, k, v, g = make(B, Lq, keys, H, H, D, dtype, seed=keys)
    q = torch.zeros_like(q)
    steps = torch.randint(-2, 3, v.shape, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    v = (v[:, :1].double() * (1 + 2 * u * steps)).to(dtype)
    out, rest, lse = dense_attention_forward(q, k, v, scale=scale, algo=algo)
    _, want, _, _, _ = definition(q, k * (scale * D ** 0.5), v, g)
    kd, vd, gd = (t.double().permute(0, 2, 1, 3) for t in (k, v, g))
    dp = gd @ vd.transpose(-1, -2)
    size = gd.abs() @ vd.abs().transpose(-1, -2)                                   # sums of magnitudes of dp, and of the row sum
    ds = (dp - dp.mean(-1, keepdim=True)) / keys
    e_ds = u * ds.abs() + (2 * (D + 2) * w + u * u + 2.0 ** -20) * (size + size.mean(-1, keepdim=True)) / keys + tiny
    tol = (scale * (e_ds @ kd.abs() + (keys + 2) * w * (ds.abs() @ kd.abs()))).permute(0, 2, 1, 3) + u * want.abs() + tiny
    dq = dense_attention_backward(q, k, v, out, rest, lse, g, scale=scale, algo=algo)[0].double()
    assert ((dq - want).abs() <= tol).all()
    without = dense_attention_backward(q, k, v, out, None, lse, g, scale=scale, algo=algo)[0].double()
    assert float(((without - want).abs() / tol).max()) > 4.0


@pytest.mark.parametrize("kind", ["rows", "ranges", "paged", "paged ranges"])
@pytest.mark.parametrize("algo", [1, 2])
def test_float16_keeps_many_small_weights_next_to_a_large_one(kind, algo):
    """One key with score 0 and the value 0, and 100000 others 17.6 below it with the value 1: each weighs 2^-25.4 of the first, less
    than float16 holds, all of them 2.3e-3.  A weight may be off by 2^-32 of the largest; the result is rounded once."""
    n, sink, u = 100001, 130, 2.0 ** -11
    rows = 300 if kind == "rows" else 3
    heads = 80 if kind == "rows" else 2
    q = torch.zeros(1, rows, heads, 64, dtype=torch.float16, device="cuda")
    q[..., 0] = 1
    k = torch.zeros(1, n, 1, 64, dtype=torch.float16, device="cuda")
    k[..., 0] = -17.59375
    v = torch.ones_like(k)
    k[:, sink, :, 0], v[:, sink] = 0, 0
    small = (n - 1) * math.exp(-17.59375)
    want = small / (1 + small)
    if kind.startswith("paged"):
        pages = -(-n // 64)
        kp, vp = (torch.cat([t[0], t[0, :pages * 64 - n]]).view(pages, 64, 1, 64) for t in (k, v))
        out = paged_attention_decode(q[:, 0], kp, vp, torch.arange(pages, dtype=torch.int32, device="cuda").view(1, -1),
                                     torch.tensor([n], dtype=torch.int32, device="cuda"), scale=1.0, algo=algo, splits=1 if kind == "paged" else 40)
    else:
        out = cross_attention(q, k, v, scale=1.0, algo=algo)
    assert float((out.double() - want).abs().max()) <= n * 2.0 ** -32 + want * (u + 2.0 ** -15)


@pytest.mark.parametrize("case", [(2, 150, 300, 4, 2, 64, torch.bfloat16), (1, 20, 5000, 2, 1, 128, torch.float16), (1, 5000, 70, 2, 2, 64, torch.bfloat16),
                                  (2, 40, 90, 2, 1, 40, torch.float32), (1, 10, 4000, 2, 2, 32, torch.float32), (2, 3, 0, 2, 2, 64, torch.float32)])
def test_gradients_that_nobody_asked_for_are_not_computed(case):
    """Each subset of the inputs gets the bits that it gets with all of them, and the entry takes null pointers for a side left out."""
    *shape, dtype = case
    q, k, v, g = make(*shape, dtype, seed=8)
    want = run_training(q, k, v, g, algo=0)
    for subset in ((0,), (1,), (2,), (1, 2), (0, 2)):
        leaves = [t.detach().requires_grad_(i in subset) for i, t in enumerate((q, k, v))]
        with torch.autograd.graph.save_on_cpu():                 # and what is saved may be stored elsewhere meanwhile
            out = cross_attention(*leaves)
        made = torch.autograd.grad(out, [leaves[i] for i in subset], g)
        assert all(torch.equal(a, want[i]) for a, i in zip(made, subset))
    if shape[2]:
        out, rest, lse = dense_attention_forward(q, k, v, scale=shape[-1] ** -0.5)
        dq, dk, dv = dense_attention_backward(q, k, v, out, rest, lse, g, scale=shape[-1] ** -0.5, need_kv=False)
        assert dk is None and dv is None and torch.equal(dq, want[0])
        dq, dk, dv = dense_attention_backward(q, k, v, out, rest, lse, g, scale=shape[-1] ** -0.5, need_q=False)
        assert dq is None and torch.equal(dk, want[1]) and torch.equal(dv, want[2])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", [120.0, 1000.0, 4096.0, 30000.0])
def test_scores_so_large_that_their_rounding_shows(size, dtype):
    """Every score 1.2e5, 8e6, 1.3e8, 7e9: the 32-bit log-sum-exp is then off by a part of 1, or by tens (its tolerance says by how much),
    and a weight recomputed from it passes 1.  Results stay finite, and the forward stays the mean of the values."""
    q, k, v, g = make(1, 130, 300, 1, 1, 64, dtype, seed=14)
    q, k = torch.full_like(q, size), torch.full_like(k, size)
    out, *grads = check(q, k, v, g, algo=2)
    assert all(t.isfinite().all() for t in grads)
    mean = v[0, :, 0].double().mean(0)
    u = torch.finfo(dtype).eps / 2
    assert ((out[0, :, 0].double() - mean).abs() <= u * mean.abs() + (u + 2.0 ** -15) * v[0, :, 0].double().abs().mean(0)).all()
    page = torch.arange(19, dtype=torch.int32, device="cuda").view(1, -1)
    kp, vp = (torch.cat([t[0], t[0, :4]]).view(19, 16, 1, 64) for t in (k, v))
    got = paged_attention_decode(q[:, 0], kp, vp, page, torch.tensor([300], dtype=torch.int32, device="cuda"), algo=2)
    assert ((got[0, 0].double() - mean).abs() <= u * mean.abs() + (u + 2.0 ** -15) * v[0, :, 0].double().abs().mean(0)).all()


@pytest.mark.parametrize("algo", [1, 2])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_large_scores_of_either_sign_choose_the_largest(dtype, algo):
    """Scores from -7e9 to 7e9 in steps that no rounding closes: the result is the one value, row by row, wherever its key lies."""
    Lq, Lk = 140, 330
    q, _, v, _ = make(1, Lq, Lk, 1, 1, 64, dtype, seed=4)
    order = torch.randperm(Lk, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    k = torch.zeros_like(v)
    k[0, :, 0, 0] = ((order.double() + 1) * 64 - 10624).to(dtype)                       # at least 64 apart in float16, 0 to 128 in bfloat16
    q = torch.zeros_like(q)
    q[0, :, 0, 0] = torch.linspace(-30000, 30000, Lq, device="cuda").to(dtype)
    out, _, lse = dense_attention_forward(q, k, v, scale=8.0, algo=algo)
    s = 8 * q[0, :, 0, 0].double().view(-1, 1) * k[0, :, 0, 0].double()
    p = torch.softmax(s, -1)
    want = p @ v[0, :, 0].double()
    u = torch.finfo(dtype).eps / 2
    assert ((out[0, :, 0].double() - want).abs() <= (u + 2.0 ** -15) * (p @ v[0, :, 0].double().abs()) + u * want.abs()).all()
    top = s.amax(-1) + torch.log(torch.exp(s - s.amax(-1, keepdim=True)).sum(-1))
    assert ((lse[0, :, 0].double() - top).abs() <= (top.abs() + 4) * 2.0 ** -22).all()


def test_float16_training_captured_and_replayed():
    """The powers of two follow each replay's own inputs, up and down, and two graphs do not disturb each other."""
    shapes = [(2, 140, 300, 4, 2, 64), (1, 20, 5000, 2, 2, 128)]
    static, graphs = [], []
    for shape in shapes:
        static.append([t.clone() for t in make(*shape, torch.float16, seed=3)])
        run_training(*static[-1], algo=0)
    torch.cuda.synchronize()
    for tensors in static:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = run_training(*tensors, algo=0)
        graphs.append((graph, res))
    for seed, size in ((5, 1e-3), (6, 4.0), (7, 1e-4), (8, 0.0)):
        for tensors, shape in zip(static, shapes):
            for t, new in zip(tensors, make(*shape, torch.float16, seed=seed)):
                t.copy_(new)
            tensors[3].mul_(size)
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for tensors, (_, res) in zip(static, graphs):
            assert all(torch.equal(a, b) for a, b in zip(res, run_training(*tensors, algo=0)))
            _, *want, _ = definition(*tensors)
            for name, a, b in zip(("dq", "dk", "dv"), res, want):
                assert not a.any() if size == 0 else as_good_as_rounded(a, b, name) is None


def test_float16_small_gradients_next_to_large_ones():
    """Output gradients of 30 over sharp weights: entries of dk range from 20 down to what float16 does not hold, and none may be off by
    more than the rounding of a score gradient as it is, half of 2^-24, would make it."""
    for shape, scale in (((1, 4, 89, 1, 1, 128), 0.3), ((2, 1, 973, 2, 2, 96), 96 ** -0.5)):
        q, k, v, g = make(*shape, torch.float16, seed=3, sharp=3.0)
        check(q, k, v, (g.float() * 30).half(), scale=scale, algo=2)
