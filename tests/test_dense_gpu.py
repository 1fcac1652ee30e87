"""Dense attention (cross_attention, paged_attention_decode) against its definition in 64 bits.

Tolerances are derived, entry by entry, from how often a value is rounded.  With u = eps / 2 of the type of the tensors (half a
step) and w = 2^-24 (half a step of the 32-bit arithmetic):
  * a score q.k is a sum of D products in 32 bits: off by at most (D + 2) w |q||k|; the logarithm of the sum inherits that;
  * the exponential and its argument add (|score| + |lse| + 4) 2^-22 relative;
  * on the tensor cores a weight, and a gradient of a score, is rounded once to the type (and below 2^-14 a float16 number is off
    by up to 2^-25 absolute);
  * a sum of n terms in 32 bits is off by at most n w times the sum of their magnitudes (taken as 2 sqrt(n) + 8: the sums are over
    independent signs, and blocked);
  * the result is rounded once to the type, and the stored output enters the row sums of the backward with that rounding.
"""
import math

import pytest
import torch

from sparseattention_b200 import HierarchicalAttention, _lib
from sparseattention_b200.ops import cross_attention, paged_attention_decode
from sparseattention_b200.ops.dense import dense_aborts, dense_attention_backward, dense_attention_forward
from tests.conftest import rel_err

pytestmark = pytest.mark.gpu

W = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
ABS_STEP = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}


def heads_first(t, heads):
    """[B, n, Hk, D] -> [B, heads, n, D] in 64 bits, shared heads repeated."""
    t = t.detach().double().permute(0, 2, 1, 3)
    return t.repeat_interleave(heads // t.size(1), dim=1)


class Definition:
    """Value, gradients and tolerances of attention over the pairs in `allowed` [B, H or 1, Lq or 1, Lk]."""

    def __init__(self, q, k, v, allowed=None, dout=None, scale=None, empty_value=0.0):
        B, Lq, H, D = q.shape
        Lk, Hkv = k.size(1), k.size(2)
        scale = D ** -0.5 if scale is None else scale
        u, tiny = HALF_STEP[q.dtype], ABS_STEP[q.dtype]
        allowed = torch.ones(1, 1, 1, 1, dtype=torch.bool, device=q.device) if allowed is None else allowed
        allowed = allowed.expand(B, H, Lq, Lk)
        seen = allowed.any(dim=2)                                        # keys nobody sees may hold anything
        qd, kd, vd = heads_first(q, H), heads_first(k, H), heads_first(v, H)
        kd, vd = torch.where(seen.unsqueeze(-1), kd, 0.0), torch.where(seen.unsqueeze(-1), vd, 0.0)
        s = scale * qd @ kd.transpose(-1, -2)
        s = s.masked_fill(~allowed, -math.inf)
        top = s.amax(dim=-1, keepdim=True)
        none = top == -math.inf
        e = torch.exp(s - torch.where(none, 0.0, top))
        total = e.sum(dim=-1, keepdim=True)
        p = torch.where(none, 0.0, e / torch.where(none, 1.0, total))
        out = p @ vd
        lse = torch.where(none, -math.inf, top + torch.log(torch.where(none, 1.0, total)))
        # how far the weights may be off
        n_sum = lambda n: (2.0 * math.sqrt(n) + 8.0) * W                                                    # noqa: E731
        ds_dot = (D + 2) * W * scale * (qd.norm(dim=-1).unsqueeze(-1) * kd.norm(dim=-1).unsqueeze(-2))
        ds_dot = torch.where(allowed, ds_dot, 0.0)
        off = ds_dot + ds_dot.amax(dim=-1, keepdim=True) + (torch.where(allowed, s.abs(), 0.0) + torch.where(none, 0.0, lse.abs()) + 4) * 2.0 ** -22
        ep = p * (u + off + n_sum(Lk)) + torch.where(none, 0.0, tiny)      # weights relative to the row's maximum: at most 1
        va = vd.abs()
        self.out = torch.where(none, empty_value, out).permute(0, 2, 1, 3)
        self.out_tol = (ep @ va + n_sum(Lk) * (p @ va) + u * out.abs() + tiny).permute(0, 2, 1, 3)
        self.lse = lse.squeeze(-1).permute(0, 2, 1)
        self.lse_tol = (ds_dot.amax(dim=-1) + (lse.squeeze(-1).nan_to_num(neginf=0.0).abs() + 4) * 2.0 ** -22 + n_sum(Lk)).permute(0, 2, 1)
        if dout is None:
            return
        g = heads_first(dout, H)
        ga = g.abs()
        sum_heads = lambda t: t.view(B, Hkv, H // Hkv, Lk, D).sum(dim=2).permute(0, 2, 1, 3)                 # noqa: E731
        back = lambda t: t.permute(0, 2, 1, 3)                                                               # noqa: E731
        dp = g @ vd.transpose(-1, -2)
        delta = (g * out).sum(dim=-1, keepdim=True)
        ds = p * (dp - delta)
        e_dp = (D + 2) * W * (ga @ va.transpose(-1, -2)) + (u + (D + 2) * W) * (ga * out.abs()).sum(-1, keepdim=True) \
            + (ga * (ep @ va)).sum(-1, keepdim=True)
        e_ds = ds.abs() * u + p * e_dp + (dp - delta).abs() * p * (off + n_sum(Lk)) + torch.where(allowed & ~none, tiny, 0.0)
        ka, qa = kd.abs(), qd.abs()
        self.dq = back(scale * ds @ kd)
        self.dq_tol = back(scale * (e_ds @ ka + n_sum(Lk) * (ds.abs() @ ka))) + u * self.dq.abs() + tiny
        n_q = n_sum(Lq * H // Hkv)
        self.dk = sum_heads(scale * ds.transpose(-1, -2) @ qd)
        self.dk_tol = sum_heads(scale * (e_ds.transpose(-1, -2) @ qa + n_q * (ds.abs().transpose(-1, -2) @ qa))) + u * self.dk.abs() + tiny
        self.dv = sum_heads(p.transpose(-1, -2) @ g)
        epv = p * (u + off + n_sum(Lk)) + torch.where(allowed & ~none, tiny, 0.0)
        self.dv_tol = sum_heads(epv.transpose(-1, -2) @ ga + n_q * (p.transpose(-1, -2) @ ga)) + u * self.dv.abs() + tiny


def near(got, want, tol, what):
    got = got.detach().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(torch.isfinite(got), torch.isfinite(want)), f"{what}: finite in other places"
    diff = torch.where(torch.isfinite(want), (got - want).abs(), 0.0)
    worst = (diff / tol.clamp_min(1e-300)).amax() if diff.numel() else torch.tensor(0.0)
    assert float(worst) <= 1.0, f"{what}: off by {float(worst):.3g} times the tolerance (largest difference {float(diff.amax()):.3g})"


def make(B, Lq, Lk, H, Hkv, D, dtype, seed=0, sharp=1.5):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda")                                            # noqa: E731
    return ((rnd(B, Lq, H, D) * sharp).to(dtype), rnd(B, Lk, Hkv, D).to(dtype), rnd(B, Lk, Hkv, D).to(dtype), rnd(B, Lq, H, D).to(dtype))


def by_length(lengths, Lk):
    return (torch.arange(Lk, device="cuda") < lengths.view(-1, 1)).view(-1, 1, 1, Lk)


def check(q, k, v, g, key_lengths=None, mask=None, scale=None, algo=0, empty_value=0.0):
    Lk = k.size(1)
    allowed = None
    if key_lengths is not None:
        allowed = by_length(key_lengths, Lk)
    if mask is not None:
        m4 = (mask != 0) if mask.dim() == 4 else (mask != 0).view(1, 1, *mask.shape)
        allowed = m4 if allowed is None else allowed & m4
    want = Definition(q, k, v, allowed, g, scale, empty_value)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = cross_attention(*leaves, key_lengths=key_lengths, mask=mask, scale=scale, empty_value=empty_value, algo=algo)
    near(out, want.out, want.out_tol, "out")
    with torch.no_grad():
        assert torch.equal(cross_attention(q, k, v, key_lengths=key_lengths, mask=mask, scale=scale, empty_value=empty_value, algo=algo)
                           .nan_to_num(7.0), out.nan_to_num(7.0))
    dq, dk, dv = torch.autograd.grad(out, leaves, g)
    near(dq, want.dq, want.dq_tol, "dq")
    near(dk, want.dk, want.dk_tol, "dk")
    near(dv, want.dv, want.dv_tol, "dv")
    return out, dq, dk, dv


SHAPES = [(1, 1, 1, 1, 1, 8), (2, 3, 5, 2, 1, 10), (1, 16, 77, 8, 8, 64), (2, 130, 129, 4, 2, 64), (1, 128, 128, 2, 2, 32),
          (2, 257, 300, 4, 4, 128), (3, 65, 127, 6, 2, 96), (1, 300, 1000, 2, 2, 80), (2, 33, 70, 2, 1, 256), (1, 5, 20, 3, 1, 200),
          (2, 1, 259, 4, 4, 64), (1, 513, 1, 2, 1, 128), (1, 40, 6000, 2, 1, 64), (1, 5000, 70, 4, 2, 128), (1, 70, 640, 3, 3, 24), (1, 256, 385, 8, 1, 72), (2, 64, 64, 1, 1, 17)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("algo", [1, 0])
def test_attention(shape, dtype, algo):
    check(*make(*shape, dtype, seed=sum(shape)), algo=algo)


@pytest.mark.parametrize("shape", [s for s in SHAPES if s[0] > 1] + [(7, 140, 390, 2, 2, 64), (6, 200, 513, 4, 2, 128)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_key_lengths(shape, dtype, index):
    B, Lk = shape[0], shape[2]
    lengths = torch.tensor([Lk, 0, 1, Lk // 2, Lk - 1, 128, Lk + 5][:B], dtype=index, device="cuda")
    q, k, v, g = make(*shape, dtype, seed=1)
    for b in range(B):                                     # what lies behind a length reaches nothing
        k[b, int(lengths[b]):] = math.nan
        v[b, int(lengths[b]):] = math.inf
    out, dq, dk, dv = check(q, k, v, g, key_lengths=lengths)
    assert not out[1].any() and not dq[1].any() and not dk[1].any() and not dv[1].any()


def test_lengths_outside_the_rows_mean_the_nearer_end():
    q, k, v, g = make(4, 20, 140, 2, 2, 64, torch.bfloat16)
    wild = torch.tensor([-3, 141, 2 ** 40, -2 ** 40], device="cuda")
    near_end = torch.tensor([0, 140, 140, 0], device="cuda")
    assert torch.equal(cross_attention(q, k, v, key_lengths=wild), cross_attention(q, k, v, key_lengths=near_end))
    wild32 = torch.tensor([-2 ** 31, 141, 2 ** 31 - 1, -1], dtype=torch.int32, device="cuda")
    assert torch.equal(cross_attention(q, k, v, key_lengths=wild32), cross_attention(q, k, v, key_lengths=near_end))


def some_mask(kind, B, H, Lq, Lk, seed=3):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if kind == "keys":
        m = torch.rand(B, 1, 1, Lk, generator=gen, device="cuda") < 0.6
        m[0, ..., : min(130, Lk // 2)] = False              # whole tiles gone
        return m
    if kind == "queries":
        m = torch.rand(1, 1, Lq, Lk, generator=gen, device="cuda") < 0.5
        m[:, :, Lq // 3] = False                            # rows that see nothing
        m[:, :, -1] = False
        return m
    if kind == "heads":
        return torch.rand(B, H, Lq, Lk, generator=gen, device="cuda") < 0.3
    if kind == "packed":
        m = torch.zeros(B, 1, Lq, Lk, dtype=torch.bool, device="cuda")
        m[:, :, : Lq // 2, : Lk // 3] = True
        m[:, :, Lq // 2: Lq - 2, Lk // 3: max(Lk - 7, 0)] = True
        return m
    if kind == "causal":
        return torch.ones(Lq, Lk, device="cuda").tril(Lk - Lq).to(torch.int32)
    if kind == "nothing":
        return torch.zeros(1, 1, 1, Lk, dtype=torch.uint8, device="cuda")
    return torch.ones(1, 1, Lq, 1, dtype=torch.int64, device="cuda") * 256         # the low byte of every entry is zero


@pytest.mark.parametrize("kind", ["keys", "queries", "heads", "packed", "causal", "nothing", "all"])
@pytest.mark.parametrize("shape", [(2, 130, 300, 4, 2, 64), (1, 300, 257, 2, 2, 128), (2, 5, 40, 2, 1, 32), (2, 140, 200, 2, 2, 20), (1, 1, 300, 2, 2, 64)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_masks(kind, shape, dtype):
    B, Lq, Lk, H, _, _ = shape
    q, k, v, g = make(*shape, dtype, seed=5)
    check(q, k, v, g, mask=some_mask(kind, B, H, Lq, Lk))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_mask_together_with_lengths_and_garbage_in_hidden_keys(dtype):
    q, k, v, g = make(3, 150, 400, 4, 2, 64, dtype, seed=6)
    lengths = torch.tensor([400, 131, 0], dtype=torch.int32, device="cuda")
    for kind in ("packed", "keys"):
        mask = some_mask(kind, 3, 4, 150, 400)
        hidden = ~mask.any(dim=2).any(dim=1)                # keys that no query looks at
        k2, v2 = k.clone(), v.clone()
        k2[hidden] = math.nan
        v2[hidden] = math.inf
        check(q, k2, v2, g, key_lengths=lengths, mask=mask)


def test_mask_strides_and_broadcast_are_those_of_the_tensor():
    q, k, v, g = make(2, 70, 150, 2, 2, 64, torch.bfloat16, seed=7)
    base = torch.rand(150, 70, device="cuda") < 0.5
    mask = base.t()                                          # keys strided, queries contiguous
    a = cross_attention(q, k, v, mask=mask)
    b = cross_attention(q, k, v, mask=mask.contiguous())
    c = cross_attention(q, k, v, mask=mask.view(1, 1, 70, 150).expand(2, 2, 70, 150))
    d = cross_attention(q, k, v, mask=torch.stack([mask, mask])[:, None].to(torch.int64) * -5)
    assert torch.equal(a, b) and torch.equal(a, c) and torch.equal(a, d)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_rows_without_keys_take_the_empty_value_and_pass_no_gradient(dtype):
    q, k, v, g = make(2, 40, 60, 2, 2, 64, dtype)
    lengths = torch.tensor([0, 60], dtype=torch.int32, device="cuda")
    out, dq, dk, dv = check(q, k, v, g, key_lengths=lengths, empty_value=math.nan)
    assert out[0].isnan().all() and not out[1].isnan().any()
    for t in (dq, dk, dv):
        assert t.isfinite().all() and not t[0].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_no_queries_no_keys_no_batch(dtype):
    for B, Lq, Lk in ((0, 4, 5), (2, 0, 5), (2, 4, 0)):
        q, k, v, g = make(B, Lq, Lk, 2, 2, 64, dtype)
        leaves = [t.requires_grad_(True) for t in (q, k, v)]
        out = cross_attention(*leaves, empty_value=3.0, mask=torch.ones(Lq, Lk, dtype=torch.bool, device="cuda"))
        assert out.shape == q.shape and (out == 3.0).all()
        for t, grad in zip(leaves, torch.autograd.grad(out, leaves, g)):
            assert grad.shape == t.shape and not grad.any()


@pytest.mark.parametrize("D", [64, 128, 40])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_shared_and_unaligned_inputs(D, dtype):
    B, Lq, Lk, H = 2, 150, 200, 4
    gen = torch.Generator(device="cuda").manual_seed(9)
    stacked = torch.randn(B, Lk, 2, H, D, generator=gen, device="cuda").to(dtype)
    k, v = stacked.unbind(dim=2)                             # strided rows
    q = torch.randn(Lq, B, H, D, generator=gen, device="cuda").to(dtype).transpose(0, 1)
    g = torch.randn(B, H, Lq, D, generator=gen, device="cuda").to(dtype).transpose(1, 2)       # heads not packed inside a row
    check(q, k, v, g)
    check(q, k[:1].expand(B, Lk, H, D), v[:1].expand(B, Lk, H, D), g)                          # one memory for the whole batch
    check(q, k[:, :1].expand(B, Lk, H, D), v, g)                                               # one key row
    flat = torch.randn(B * Lq * H * D + 1, generator=gen, device="cuda").to(dtype)
    check(flat[1:].view(B, Lq, H, D), k, v, g)                                                 # not 16-byte aligned
    check(q[:, ::3], k[:, 1::2], v[:, 1::2], g[:, ::3])
    check(q, k, v, g[:1, :1].expand(B, Lq, H, D))


def test_broadcast_inputs_get_summed_gradients():
    q, k, v, g = make(3, 40, 50, 2, 2, 64, torch.float32, seed=11)
    k1, v1 = k[:1].clone().requires_grad_(True), v[:1].clone().requires_grad_(True)
    out = cross_attention(q, k1.expand(3, -1, -1, -1), v1.expand(3, -1, -1, -1))
    dk, dv = torch.autograd.grad(out, (k1, v1), g)
    want = Definition(q, k[:1].expand(3, -1, -1, -1), v[:1].expand(3, -1, -1, -1), None, g)
    near(dk, want.dk.sum(0, keepdim=True), want.dk_tol.sum(0, keepdim=True), "dk")
    near(dv, want.dv.sum(0, keepdim=True), want.dv_tol.sum(0, keepdim=True), "dv")


def test_gradients_against_differences():
    """Central differences of a random projection of the output, step h: the quotient is off by h^2 / 6 times a third derivative
    (of order one here, with entries of order one) plus twice the output's rounding over 2 h."""
    q, k, v, g = make(1, 6, 9, 2, 1, 16, torch.float32, seed=12, sharp=1.0)
    mask = torch.rand(6, 9, device="cuda") < 0.7
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(cross_attention(*leaves, mask=mask), leaves, g)
    gen = torch.Generator(device="cuda").manual_seed(4)
    h = 1e-2
    for i, grad in enumerate(grads):
        for _ in range(4):
            d = torch.randn(leaves[i].shape, generator=gen, device="cuda")
            d = d / d.norm()
            f = []
            for s in (h, -h):
                moved = [t.detach() + (s * d if j == i else 0) for j, t in enumerate(leaves)]
                f.append(float((cross_attention(*moved, mask=mask).double() * g.double()).sum()))
            quotient, slope = (f[0] - f[1]) / (2 * h), float((grad.double() * d.double()).sum())
            rounding = 2 * float(g.abs().sum()) * 4 * 2.0 ** -22 / (2 * h)
            assert abs(quotient - slope) <= h * h * float(g.norm()) + rounding, (i, quotient, slope)


@pytest.mark.parametrize("scale", [1.0, 0.01, 0.5])
def test_scale(scale):
    for dtype in (torch.float32, torch.float16):
        check(*make(2, 70, 150, 2, 2, 64, dtype, sharp=0.3), scale=scale)


def test_scores_of_large_and_falling_size():
    """A maximum that moves by hundreds from tile to tile, up and down, and weights that vanish."""
    for sign in (1.0, -1.0):
        q, k, v, g = make(1, 140, 700, 2, 2, 64, torch.bfloat16, seed=13)
        k *= torch.linspace(0.1, 8.0, 700, device="cuda").view(1, -1, 1, 1).to(k.dtype) if sign > 0 else \
            torch.linspace(8.0, 0.1, 700, device="cuda").view(1, -1, 1, 1).to(k.dtype)
        check(q, k, v, g)
    q, k, v, g = make(1, 130, 300, 1, 1, 64, torch.bfloat16, seed=14)
    check(torch.full_like(q, 30.0), torch.full_like(k, 30.0), v, g)          # every score 7200


def test_nan_and_infinite_scores_show():
    q, k, v, g = make(1, 130, 300, 2, 2, 64, torch.bfloat16)
    q[0, 5, 1] = math.nan
    out = cross_attention(q, k, v)
    assert out[0, 5, 1].isnan().all()
    out[0, 5, 1] = 0
    assert out.isfinite().all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_two_runs_give_the_same_bits(dtype):
    q, k, v, g = make(2, 300, 500, 8, 2, 64, dtype)
    mask = some_mask("queries", 2, 8, 300, 500)
    runs = []
    for _ in range(2):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = cross_attention(*leaves, mask=mask)
        runs.append((out.detach(), *torch.autograd.grad(out, leaves, g)))
    assert all(torch.equal(a, b) for a, b in zip(*runs))


@pytest.mark.parametrize("shape", [(2, 140, 300, 4, 2, 64), (1, 20, 5000, 2, 2, 128), (2, 1, 700, 4, 4, 64)])
def test_capture_and_replay_on_new_inputs_and_other_streams(shape):
    q, k, v, g = make(*shape, torch.bfloat16, seed=15)
    q2, k2, v2, g2 = make(*shape, torch.bfloat16, seed=16)
    Lk = shape[2]
    lengths = torch.full((shape[0],), Lk, dtype=torch.int32, device="cuda")
    static = [t.clone() for t in (q, k, v)]
    gs = g.clone()

    def step():
        leaves = [t.detach().requires_grad_(True) for t in static]
        out = cross_attention(*leaves, key_lengths=lengths)
        return (out.detach(), *torch.autograd.grad(out, leaves, gs))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = step()
        graphs.append((graph, res))
    for graph, res in graphs:
        graph.replay()
    torch.cuda.synchronize()
    for _, res in graphs:
        assert all(torch.equal(a, b) for a, b in zip(res, eager))
    for s, t in zip(static, (q2, k2, v2)):
        s.copy_(t)
    gs.copy_(g2)
    lengths.fill_(max(1, Lk // 2))
    for graph, _ in graphs:
        graph.replay()
    torch.cuda.synchronize()
    want = step()
    for _, res in graphs:
        assert all(torch.equal(a, b) for a, b in zip(res, want))


@pytest.mark.parametrize("shape,rows", [((1, 3, 98500, 2, 2, 64), 1), ((1, 50000, 10, 2, 1, 64), 50000)])
def test_masks_beyond_the_tile_table(shape, rows):
    """More 128 x 128 cells along one side than the tensor-core kernels keep per block: the 32-bit kernels take over."""
    B, Lq, Lk, H, Hkv, D = shape
    q, k, v, g = make(*shape, torch.bfloat16, seed=17)
    mask = torch.rand(1, 1, rows, Lk, device="cuda") < 0.5
    check(q, k, v, g, mask=mask)


def test_offsets_past_32_bits():
    """Keys and values of more than 2^31 elements, zeros but for the last rows: every zero row scores 0 and adds nothing."""
    Lk, H, D, tail, Lq = 2_200_000, 8, 128, 300, 5
    assert Lk * H * D > 2 ** 31
    q, kt, vt, g = make(1, Lq, tail, H, H, D, torch.bfloat16, seed=18)
    k = torch.zeros(1, Lk, H, D, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros(1, Lk, H, D, dtype=torch.bfloat16, device="cuda")
    k[:, -tail:], v[:, -tail:] = kt * 3, vt
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = cross_attention(*leaves)
    dq, dk, dv = torch.autograd.grad(out, leaves, g)
    qd, kd, vd, gd = (heads_first(t, H) for t in (q, kt * 3, vt, g))
    s = D ** -0.5 * qd @ kd.transpose(-1, -2)
    top = s.amax(dim=-1, keepdim=True).clamp_min(0.0)
    total = torch.exp(s - top).sum(dim=-1, keepdim=True) + (Lk - tail) * torch.exp(-top)
    p = torch.exp(s - top) / total
    o = p @ vd
    ds = p * (gd @ vd.transpose(-1, -2) - (gd * o).sum(-1, keepdim=True))
    flat = -torch.exp(-top) / total * (gd * o).sum(-1, keepdim=True)          # ds of a zero row
    back = lambda t: t.permute(0, 2, 1, 3)                                      # noqa: E731
    for name, got, want in (("out", out, back(o)), ("dv", dv[:, -tail:], back(p.transpose(-1, -2) @ gd)),
                            ("dk", dk[:, -tail:], back(D ** -0.5 * ds.transpose(-1, -2) @ qd)), ("dq", dq, back(D ** -0.5 * ds @ kd)),
                            ("dk of a zero row", dk[:, :2], back(D ** -0.5 * (flat * qd).sum(2, keepdim=True)).expand(1, 2, H, D))):
        assert rel_err(got.detach().double(), want) < 2e-2, name


def test_log_sum_exp():
    for dtype in (torch.float32, torch.bfloat16):
        q, k, v, _ = make(2, 70, 300, 4, 2, 64, dtype)
        lengths = torch.tensor([300, 0], dtype=torch.int32, device="cuda")
        want = Definition(q, k, v, by_length(lengths, 300))
        _, _, lse = dense_attention_forward(q, k, v, lengths, None, 64 ** -0.5)
        near(lse, want.lse, want.lse_tol, "lse")


def test_refusals():
    q, k, v, _ = make(2, 4, 6, 2, 2, 64, torch.bfloat16)
    with pytest.raises(_lib.HsaError):
        cross_attention(q, k, v, mask=torch.zeros(4, 6, device="cuda"))                   # an additive mask
    with pytest.raises(AssertionError):
        cross_attention(q, k, v, mask=torch.ones(2, 4, 6, dtype=torch.bool, device="cuda"))
    with pytest.raises(AssertionError):
        cross_attention(q, k, v, mask=torch.ones(4, 5, dtype=torch.bool, device="cuda"))
    with pytest.raises(_lib.HsaError):
        cross_attention(q, k, v, mask=torch.ones(4, 6, dtype=torch.bool))                 # on the host
    with pytest.raises(_lib.HsaError):
        cross_attention(q, k, v, key_lengths=torch.ones(2, device="cuda"))
    with pytest.raises(AssertionError):
        cross_attention(q, k, v, key_lengths=torch.ones(3, dtype=torch.int32, device="cuda"))
    with pytest.raises(AssertionError):
        cross_attention(q, k.float(), v.float())
    with pytest.raises(AssertionError):
        cross_attention(q, k[:, :5], v)
    with pytest.raises(AssertionError):
        cross_attention(q[:, :, :1].expand(2, 4, 3, 64), k, v)
    with pytest.raises(_lib.HsaError):
        cross_attention(q.double(), k.double(), v.double())
    for scale in (0.0, -0.1, math.nan, math.inf):
        with pytest.raises(_lib.HsaError):
            cross_attention(q, k, v, scale=scale)
    with pytest.raises(_lib.HsaError):
        cross_attention(q.float(), k.float(), v.float(), algo=2)                          # float32 has no tensor-core kernel
    leaf = q.clone().requires_grad_(True)
    (grad,) = torch.autograd.grad(cross_attention(leaf, k, v).float().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(grad.float().sum(), leaf)


# ---------------------------------------------------------------------------------------------------------------- paged
def make_cache(B, H, Hkv, D, page, lengths, dtype, seed=0, spare=3, width=None):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    need = [-(-n // page) for n in lengths]
    width = max(1, max(need)) if width is None else width
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")       # entries behind a length are never read
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    q = torch.randn(B, H, D, generator=gen, device="cuda").mul(1.5).to(dtype)
    kp = torch.randn(pages, page, Hkv, D, generator=gen, device="cuda").to(dtype)
    vp = torch.randn(pages, page, Hkv, D, generator=gen, device="cuda").to(dtype)
    used = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
    for b, n in enumerate(lengths):
        for i in range(need[b]):
            used[table[b, i].long(), : min(page, n - i * page)] = True
    kp[~used] = math.nan                                                       # nor are slots behind it
    vp[~used] = math.inf
    return q, kp, vp, table, torch.tensor(lengths, dtype=torch.int32, device="cuda")


def check_paged(q, kp, vp, table, lengths, **kw):
    got = paged_attention_decode(q, kp, vp, table, lengths, **kw)
    page = kp.size(1)
    for b, n in enumerate(lengths.tolist()):
        if n == 0:
            assert not got[b].any()
            continue
        rows = table[b, : -(-n // page)].long()
        k, v = (t[rows].flatten(0, 1)[:n].unsqueeze(0) for t in (kp, vp))
        want = Definition(q[b:b + 1].unsqueeze(1), k, v)
        near(got[b].view(1, 1, *got[b].shape), want.out, want.out_tol, f"sequence {b}")
    return got


PAGED = [(1, 1, 1, 8, 1, [1]), (1, 8, 8, 64, 16, [100]), (3, 4, 2, 64, 16, [0, 1, 333]), (2, 16, 1, 128, 64, [700, 65]),
         (2, 6, 2, 96, 24, [250, 24]), (1, 24, 1, 32, 7, [500]), (2, 40, 2, 128, 32, [129, 1000]), (2, 5, 5, 256, 16, [90, 300]),
         (1, 4, 4, 10, 16, [77]), (2, 2, 1, 200, 128, [400, 3]), (1, 8, 2, 128, 256, [9000])]


@pytest.mark.parametrize("case", PAGED)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("algo", [1, 0])
@pytest.mark.parametrize("splits", [None, 1, 3, 50])
def test_paged_decode(case, dtype, algo, splits):
    B, H, Hkv, D, page, lengths = case
    check_paged(*make_cache(B, H, Hkv, D, page, lengths, dtype, seed=D), algo=algo, splits=splits)


@pytest.mark.parametrize("case", [(40, 8, 8, 64, 16), (128, 6, 3, 128, 16), (129, 3, 3, 64, 16), (65, 5, 5, 200, 32)])
@pytest.mark.parametrize("splits", [None, 1, 2])
def test_paged_many_sequences_of_unequal_length(case, splits):
    """More blocks than run at once, where the longest sequences may start first: each sequence gives what it gives alone, bit by
    bit, whatever the others' lengths (equal ones, none, ones that the table cannot hold)."""
    B, H, Hkv, D, page = case
    lengths = [(7 * i * i) % 400 for i in range(B)]
    lengths[1], lengths[-2] = 2100, 1500
    lengths[2] = lengths[3] = lengths[-1] = 300
    lengths[4] = lengths[5] = 0
    q, kp, vp, table, n = make_cache(B, H, Hkv, D, page, lengths, torch.bfloat16, seed=B)
    chosen = _lib.load().hsa_paged_attn_choose_splits(B, H, Hkv, page, table.size(1)) if splits is None else splits
    got = check_paged(q, kp, vp, table, n, splits=splits)
    for b in (0, 1, 2, 3, 4, B // 2, B - 2, B - 1):
        assert torch.equal(paged_attention_decode(q[b:b + 1], kp, vp, table[b:b + 1], n[b:b + 1], splits=chosen)[0], got[b])
    wild = n.clone()
    wild[0], wild[7], wild[8] = -1, table.size(1) * page + 1, 2 ** 31 - 1
    bad = paged_attention_decode(q, kp, vp, table, wild, splits=splits)
    others = [b for b in range(B) if b not in (0, 7, 8)]
    assert bad[[0, 7, 8]].isnan().all() and torch.equal(bad[others], got[others])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_paged_bad_pages_and_lengths_show_as_nan(dtype):
    """What the table must not hold is not followed: the sequence's output is NaN and the others are as before."""
    for splits in (1, 4):
        q, kp, vp, table, lengths = make_cache(5, 4, 2, 64, 16, [300, 40, 200, 17, 0], dtype)
        good = paged_attention_decode(q, kp, vp, table, lengths, splits=splits)
        broken, wild = table.clone(), lengths.clone()
        broken[0, 18] = kp.size(0)                 # one past the last page
        broken[1, 0] = -1
        broken[2, 3] = 2 ** 31 - 1
        wild[3] = table.size(1) * 16 + 1           # longer than the table
        wild[4] = -1
        got = paged_attention_decode(q, kp, vp, broken, lengths, splits=splits)
        assert got[:3].isnan().all() and torch.equal(got[3:], good[3:])
        got = paged_attention_decode(q, kp, vp, table, wild, splits=splits)
        assert got[3:].isnan().all() and torch.equal(got[:3], good[:3])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_paged_strided_cache(dtype):
    """Keys and values side by side in one buffer, layers between pages, a table that is a slice of a larger one."""
    q, kp, vp, table, lengths = make_cache(3, 8, 4, 64, 16, [100, 57, 16], dtype)
    both = torch.full((kp.size(0), 2, 16, 2, 4, 64), math.nan, dtype=dtype, device="cuda")
    both[:, 1, :, 0], both[:, 1, :, 1] = kp, vp
    wide = torch.full((3, table.size(1) + 5), -7, dtype=torch.int32, device="cuda")
    wide[:, 2:2 + table.size(1)] = table
    want = paged_attention_decode(q, kp, vp, table, lengths, splits=2)
    got = paged_attention_decode(q, both[:, 1, :, 0], both[:, 1, :, 1], wide[:, 2:2 + table.size(1)], lengths, splits=2)
    assert torch.equal(got, want)
    # slots that are not 16-byte aligned
    odd = torch.empty(kp.numel() + 1, dtype=dtype, device="cuda")[1:].view(kp.shape).copy_(kp)
    near(paged_attention_decode(q, odd, vp, table, lengths), *(lambda w: (w.double(), w.double().abs() * 4 * HALF_STEP[dtype] + 2 * HALF_STEP[dtype]))(want), "odd")


def test_paged_offsets_past_32_bits():
    """Pages at both ends of a cache of more than 2^32 elements."""
    pages, page, Hkv, D = 33000, 128, 8, 128
    assert pages * page * Hkv * D > 2 ** 32
    kp = torch.empty(pages, page, Hkv, D, dtype=torch.bfloat16, device="cuda")
    vp = torch.empty(pages, page, Hkv, D, dtype=torch.bfloat16, device="cuda")
    used = torch.tensor([pages - 1, 0, pages - 2, 16500], device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(2)
    for t in (kp, vp):
        t[used] = torch.randn(4, page, Hkv, D, generator=gen, device="cuda").to(torch.bfloat16)
    q = torch.randn(1, 16, D, generator=gen, device="cuda").to(torch.bfloat16)
    table = used.to(torch.int32).view(1, 4)
    for algo in (0, 1):
        check_paged(q, kp, vp, table, torch.tensor([500], dtype=torch.int32, device="cuda"), algo=algo)


def test_paged_shared_pages_and_capture():
    """Two sequences that share their first pages; a captured step follows the table and the lengths."""
    q, kp, vp, table, lengths = make_cache(2, 8, 2, 128, 32, [200, 200], torch.bfloat16)
    table[1, :3] = table[0, :3]
    want = check_paged(q, kp, vp, table, lengths)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = paged_attention_decode(q, kp, vp, table, lengths)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    lengths.copy_(torch.tensor([33, 150], dtype=torch.int32))
    table.copy_(table.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, paged_attention_decode(q, kp, vp, table, lengths))


def test_paged_refusals():
    q, kp, vp, table, lengths = make_cache(2, 4, 2, 64, 16, [20, 30], torch.bfloat16)
    with pytest.raises(AssertionError):
        paged_attention_decode(q, kp, vp, table.long(), lengths)
    with pytest.raises(AssertionError):
        paged_attention_decode(q, kp, vp, table[:1], lengths)
    with pytest.raises(AssertionError):
        paged_attention_decode(q[:, :3], kp, vp, table, lengths)
    with pytest.raises(AssertionError):
        paged_attention_decode(q, kp.float(), vp.float(), table, lengths)
    with pytest.raises(_lib.HsaError):
        paged_attention_decode(q, kp.transpose(2, 3).contiguous().transpose(2, 3), vp, table, lengths)
    with pytest.raises(_lib.HsaError):
        paged_attention_decode(q, kp, vp, table, lengths, scale=0.0)
    with pytest.raises(_lib.HsaError):
        paged_attention_decode(q, kp, vp, table, lengths, splits=0)
    assert paged_attention_decode(q[:0], kp, vp, table[:0], lengths[:0]).shape == (0, 4, 64)
    none = paged_attention_decode(q, kp, vp, table[:, :0], torch.tensor([0, 5], dtype=torch.int32, device="cuda"))
    assert not none[0].any() and none[1].isnan().all()


def test_paged_nan_scores_show():
    for splits in (1, 3):
        q, kp, vp, table, lengths = make_cache(2, 4, 2, 64, 16, [200, 30], torch.bfloat16)
        q[0, 1] = math.nan
        for algo in (0, 1):
            got = paged_attention_decode(q, kp, vp, table, lengths, splits=splits, algo=algo)
            assert got[0, 1].isnan().all()
            got[0, 1] = 0
            assert got.isfinite().all()


def test_training_then_serving_the_same_rows():
    """The operators as they are used together: a model trains on whole sequences, then serves token by token from pages."""
    B, Lq, Lk, H, Hkv, D, page = 3, 6, 150, 8, 4, 64, 16
    q, k, v, g = make(B, Lq, Lk, H, Hkv, D, torch.bfloat16, seed=21)
    lengths = torch.tensor([150, 1, 97], dtype=torch.int32, device="cuda")
    out, dq, dk, dv = check(q, k, v, g, key_lengths=lengths)
    width = -(-Lk // page)
    table = torch.randperm(B * width, device="cuda").to(torch.int32).view(B, width)
    kp = torch.zeros(B * width, page, Hkv, D, dtype=k.dtype, device="cuda")
    vp = torch.zeros_like(kp)
    pos = torch.arange(Lk, device="cuda")
    for b in range(B):
        kp[table[b, pos // page].long(), pos % page] = k[b]
        vp[table[b, pos // page].long(), pos % page] = v[b]
    want = Definition(q, k, v, by_length(lengths, Lk))
    for i in range(Lq):
        step = paged_attention_decode(q[:, i].contiguous(), kp, vp, table, lengths)
        near(step, want.out[:, i], want.out_tol[:, i], f"token {i}")


# --------------------------------------------------------------------------------------------------------------- module
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", [None, "row", "keys", "square", "empty"])
def test_module_over_another_sequence(dtype, kind):
    """HierarchicalAttention without parents: the kernel against the module's eager operations on the same weights in 32 bits
    (2e-2, what the suite grants 16-bit layers), outputs, input and weight gradients."""
    B, Lq, Lk, d, H = 2, 75, 140, 256, 4
    torch.manual_seed(5)
    layer = HierarchicalAttention(d, H, dropout=0.1).cuda().eval()
    exact = HierarchicalAttention(d, H, dropout=0.1).cuda().eval()
    layer = layer.to(dtype)
    exact.load_state_dict({n: t.float() for n, t in layer.state_dict().items()})
    gen = torch.Generator(device="cuda").manual_seed(8)
    q, m, g = (torch.randn(B, n, d, generator=gen, device="cuda").to(dtype) for n in (Lq, Lk, Lq))
    mask = {None: None, "row": torch.rand(Lk, generator=gen, device="cuda").gt(0.3),
            "keys": torch.rand(B, 1, 1, Lk, generator=gen, device="cuda").gt(0.3).float(),
            "square": torch.rand(Lq, Lk, generator=gen, device="cuda").gt(0.5).to(torch.int32),
            "empty": torch.ones(Lq, Lk, dtype=torch.bool, device="cuda")}[kind]
    if kind == "empty":
        mask[3] = False
    calls = []
    hook = layer.dropout.register_forward_hook(lambda *a: calls.append(1))         # the eager path passes its weights through it
    ql, ml = q.clone().requires_grad_(True), m.clone().requires_grad_(True)
    out = layer(ql, ml, ml, mask=mask)
    hook.remove()
    assert not calls
    qe, me = q.float().requires_grad_(True), m.float().requires_grad_(True)
    want = exact(qe, me, me, mask=mask)
    if kind == "empty":
        assert out[:, 3].isnan().all() and want[:, 3].isnan().all()
        rest = torch.arange(Lq, device="cuda") != 3
        assert rel_err(out[:, rest].float(), want[:, rest]) < 2e-2
        return
    assert rel_err(out.float(), want) < 2e-2
    got = torch.autograd.grad(out, [ql, ml, layer.Wq_x.weight, layer.Wk_x.weight, layer.Wv_x.weight, layer.out_proj_x.bias], g)
    ref = torch.autograd.grad(want, [qe, me, exact.Wq_x.weight, exact.Wk_x.weight, exact.Wv_x.weight, exact.out_proj_x.bias], g.float())
    for a, b in zip(got, ref):
        assert rel_err(a.float(), b) < 2e-2


def test_module_keeps_its_eager_path_where_the_kernel_does_not_apply():
    layer = HierarchicalAttention(64, 2, dropout=0.5).cuda().to(torch.bfloat16)
    q, m = torch.randn(2, 9, 64, device="cuda", dtype=torch.bfloat16), torch.randn(2, 13, 64, device="cuda", dtype=torch.bfloat16)
    calls = []
    layer.dropout.register_forward_hook(lambda *a: calls.append(1))
    layer(q, m, m)                                                # dropout is active
    assert len(calls) == 1
    layer.eval()
    out, weights = layer(q, m, m, return_attention=True)          # weights asked for
    assert len(calls) == 2 and weights.shape == (2, 2, 9, 13)
    near = layer(q, m, m)
    assert len(calls) == 2 and rel_err(near.float(), out.float()) < 2e-2
    layer.fused_attention = False
    assert torch.equal(layer(q, m, m), out) and len(calls) == 3
    layer.float()
    layer.fused_attention = True
    layer(q.float(), m.float(), m.float())                        # 32 bits
    assert len(calls) == 4
    with torch.autocast("cuda", dtype=torch.bfloat16):
        layer(q.float(), m.float(), m.float())
    assert len(calls) == 4


# -------------------------------------------------------------------------------------------------------- bounded waits
def test_a_wait_that_runs_out_shows():
    """Every copy completes, but the first barrier of an item expects bytes that never come: the blocks give up after a short
    limit, count themselves and leave NaN; afterwards everything is as before."""
    lib = _lib.load()
    q, k, v, g = make(2, 200, 300, 2, 2, 64, torch.bfloat16)
    out, rest, lse = dense_attention_forward(q, k, v, None, None, 0.125)
    good = (out, *dense_attention_backward(q, k, v, out, rest, lse, g, None, None, 0.125))
    torch.cuda.synchronize()
    before = dense_aborts()
    _lib.check(lib.hsa_debug_wait_test(20_000_000, 16), "hsa_debug_wait_test")
    try:
        bad, _, bad_lse = dense_attention_forward(q, k, v, None, None, 0.125)
        torch.cuda.synchronize()
        mid = dense_aborts()
        grads = dense_attention_backward(q, k, v, out, rest, lse, g, None, None, 0.125)
        torch.cuda.synchronize()
    finally:
        _lib.check(lib.hsa_debug_wait_test(2_000_000_000, 0), "hsa_debug_wait_test")
    assert mid > before and dense_aborts() > mid
    assert bad.isnan().all() and bad_lse.isnan().all()
    assert all(t.isnan().all() for t in grads)
    out, rest, lse = dense_attention_forward(q, k, v, None, None, 0.125)
    again = (out, *dense_attention_backward(q, k, v, out, rest, lse, g, None, None, 0.125))
    assert all(torch.equal(a, b) for a, b in zip(good, again))


def test_no_wait_has_run_out():
    """Sorts last in this file: the only blocks that ever gave up are those of the test above."""
    q, k, v, g = make(4, 700, 900, 8, 8, 128, torch.bfloat16)
    before = dense_aborts()
    for _ in range(5):
        check(q, k, v, g)
    assert dense_aborts() == before
