"""Dense attention kernels whose bounded waits run out, with more work items than SMs: blocks then hold items that they took over
from the grid, and no row of any of them may be left unwritten.

Every copy of these runs completes; the first barrier of an item expects bytes that never come, the wait ends after a short limit
and the kernels return by themselves.
"""
import ctypes

import pytest
import torch

from sparseattention_b200 import _lib
from sparseattention_b200.ops import dense
from sparseattention_b200.ops.dense import dense_aborts

pytestmark = pytest.mark.gpu

SENTINEL = 16384.0                                 # exact in every type, and far beyond the results below


class Call:
    """The C entries on prefilled outputs."""

    def __init__(self, B, Lq, Lk, H, Hkv, D, dtype, lengths=None, seed=0):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(dtype)                              # noqa: E731
        self.sizes, self.dtype = (B, Lq, Lk, H, Hkv, D), dtype
        self.q, self.g, self.k, self.v = rnd(B, Lq, H, D), rnd(B, Lq, H, D), rnd(B, Lk, Hkv, D), rnd(B, Lk, Hkv, D)
        self.lengths = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")

    def _common(self):
        lib, code = _lib.load(), _lib.dtype_code(self.q)
        view = lambda t: _lib.HsaView(t.data_ptr(), t.stride(0), t.stride(1))                                 # noqa: E731
        ptr = lambda t: None if t is None else ctypes.c_void_p(t.data_ptr())                                  # noqa: E731
        return lib, code, view, ptr, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)

    def _workspace(self, nbytes):
        return torch.full((max(nbytes, 256) // 4 + 64,), SENTINEL, device="cuda") if nbytes else None

    def forward(self):
        lib, code, view, ptr, stream = self._common()
        B, Lq, Lk, H, Hkv, D = self.sizes
        out, rest = (torch.full_like(self.q, SENTINEL) for _ in range(2))
        lse = torch.full((B, Lq, H), SENTINEL, device="cuda")
        need = lib.hsa_dense_attn_fwd_workspace_bytes(*self.sizes, code, 2)
        ws = self._workspace(need)
        _lib.check(lib.hsa_dense_attn_fwd(view(self.q), view(self.k), view(self.v), view(out), ptr(rest), ptr(lse), ptr(self.lengths), None, 0,
                                          0, 0, ptr(ws), need, *self.sizes, D ** -0.5, 0.0, code, 2, stream), "forward")
        torch.cuda.synchronize()
        return out, rest, lse

    def backward(self, out, rest, lse):
        lib, code, view, ptr, stream = self._common()
        D = self.sizes[-1]
        grads = [torch.full_like(t, SENTINEL) for t in (self.q, self.k, self.v)]
        need = lib.hsa_dense_attn_bwd_workspace_bytes(*self.sizes, code, 2)
        ws = self._workspace(need)
        _lib.check(lib.hsa_dense_attn_bwd(view(self.q), view(self.k), view(self.v), view(out), ptr(rest), ptr(lse), view(self.g),
                                          *(view(t) for t in grads), ptr(self.lengths), None, 0, 0, 0, ptr(ws), need, *self.sizes,
                                          D ** -0.5, code, 2, stream), "backward")
        torch.cuda.synchronize()
        return grads


def nan_or(got, want, what):
    """Every row is NaN throughout or what it should be; returns how many are NaN."""
    got, want = (t.unsqueeze(-1) if t.dim() == 3 else t for t in (got, want))
    nan = got.isnan().all(dim=-1)
    right = ((got == want) | (got.isnan() & want.isnan())).all(dim=-1)
    lost = ~(nan | right)
    assert not lost.any(), f"{what}: {int(lost.sum())} of {lost.numel()} rows are neither"
    return int(nan.sum())


# B, Lq, Lk, H, Hkv, D, lengths: items of one or two key tiles (the next item is asked for at once), of many, empty ones between others, and
# ranges of few items
CASES = [(8, 700, 200, 16, 16, 64, None), (4, 900, 1300, 16, 8, 128, None), (16, 300, 100, 16, 16, 64, [100, 0, 1, 37] * 4),
         (16, 400, 700, 8, 8, 128, [0, 700, 0, 128] * 4), (5, 200, 25600, 10, 10, 64, None), (5, 12800, 100, 10, 10, 64, None)]


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_no_row_is_left_unwritten(case, dtype):
    *sizes, lengths = case
    call = Call(*sizes, dtype, lengths)
    good = call.forward()
    good_grads = call.backward(*good)
    assert not any((t == SENTINEL).any() for t in (good[0], *good_grads))
    before = dense_aborts()
    _lib.check(_lib.load().hsa_debug_wait_test(2_000_000, 16), "hsa_debug_wait_test")
    try:
        bad = call.forward()
        mid = dense_aborts()
        grads = call.backward(*good)
        after = dense_aborts()
    finally:
        _lib.check(_lib.load().hsa_debug_wait_test(2_000_000_000, 0), "hsa_debug_wait_test")
    assert before < mid < after
    for name, got, want in zip(("out", "rest", "lse"), bad, good):
        assert nan_or(got, want, name) > 0
    for name, got, want in zip(("dq", "dk", "dv"), grads, good_grads):
        assert nan_or(got, want, name) > 0
    again = call.forward()
    assert all(torch.equal(a, b) for a, b in zip(again, good))
    assert all(torch.equal(a, b) for a, b in zip(call.backward(*good), good_grads))


def test_the_count_waits_for_calls_on_other_streams(monkeypatch):
    """Read right after a call on a stream of its own, the count has that call's blocks, and the debug check blames it and no later one."""
    call = Call(4, 300, 200, 8, 8, 64, torch.bfloat16)
    good = call.forward()
    good_grads = call.backward(*good)
    args = (call.q, call.k, call.v)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    monkeypatch.setattr(_lib, "DEBUG", True)
    with torch.cuda.stream(side):
        monkeypatch.setattr(dense, "_aborts_seen", {torch.cuda.current_device(): dense_aborts()})
        before = dense_aborts()
        _lib.check(_lib.load().hsa_debug_wait_test(20_000_000, 16), "hsa_debug_wait_test")
        try:
            with pytest.raises(_lib.HsaError, match="fwd"):
                dense.dense_attention_forward(*args, scale=64 ** -0.5)
            with pytest.raises(_lib.HsaError, match="bwd"):
                dense.dense_attention_backward(*args, *good, call.g, scale=64 ** -0.5)
        finally:
            _lib.check(_lib.load().hsa_debug_wait_test(2_000_000_000, 0), "hsa_debug_wait_test")
        assert dense_aborts() > before
        healthy = dense.dense_attention_forward(*args, scale=64 ** -0.5)
        grads = dense.dense_attention_backward(*args, *good, call.g, scale=64 ** -0.5)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((*healthy, *grads), (*good, *good_grads)))
