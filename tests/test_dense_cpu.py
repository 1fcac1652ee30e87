"""Refusals of the dense attention entry points that need no GPU."""
import ctypes

import pytest
import torch

from sparseattention_b200 import _lib
from sparseattention_b200.ops import cross_attention, paged_attention_decode

P = ctypes.c_void_p(0x1000)
V = _lib.HsaView(0x1000, 0, 0)
NULL = _lib.HsaView(0, 0, 0)


def fwd(q=V, B=1, Lq=4, Lk=4, H=2, Hkv=2, D=64, scale=0.125, dtype=1, algo=0, mask=None, sizes=(0, 0, 0), rest=None):
    return _lib.load().hsa_dense_attn_fwd(q, V, V, V, rest, None, None, mask, *sizes, None, 0, B, Lq, Lk, H, Hkv, D, scale, 0.0, dtype,
                                          algo, None)


def bwd(B=1, Lq=4, Lk=4, H=2, Hkv=2, D=64, scale=0.125, dtype=1, ws=P, nbytes=1 << 20):
    return _lib.load().hsa_dense_attn_bwd(V, V, V, V, None, P, V, V, V, V, None, None, 0, 0, 0, ws, nbytes, B, Lq, Lk, H, Hkv, D, scale,
                                          dtype, 0, None)


def paged(table=P, B=1, H=2, Hkv=2, D=64, page=16, pages=4, width=4, scale=0.125, dtype=1, splits=1, ws=None, nbytes=0, algo=0):
    return _lib.load().hsa_paged_attn_decode(V, V, V, V, table, width, P, ws, nbytes, B, H, Hkv, D, page, pages, width, scale, dtype,
                                             splits, algo, None)


@pytest.mark.parametrize("call", [fwd, bwd])
@pytest.mark.parametrize("bad", [dict(B=0), dict(Lq=0), dict(Lk=0), dict(H=3, Hkv=2), dict(Hkv=0), dict(D=0), dict(D=257),
                                 dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")), dict(scale=float("nan")),
                                 dict(Lk=(1 << 30) + 1)])
def test_attention_refuses_bad_shapes(call, bad):
    assert call(**bad) == -1
    assert _lib.load().hsa_last_error()


def test_attention_refuses_the_rest():
    assert fwd(q=NULL) == -1
    assert fwd(dtype=7) == -3 and bwd(dtype=-1) == -3
    assert fwd(algo=3) == -1
    assert fwd(rest=P, dtype=0) == -1 and fwd(rest=ctypes.c_void_p(0x1008)) == -2
    assert fwd(mask=P, sizes=(2, 1, 1), B=3) == -1 and b"broadcast" in _lib.load().hsa_last_error()
    assert fwd(mask=P, sizes=(1, 1, 3), Lq=4) == -1
    assert bwd(ws=None) == -4 and bwd(nbytes=8) == -4
    assert bwd(ws=ctypes.c_void_p(0x1010)) == -2


def test_mask_sizes():
    lib = _lib.load()
    assert lib.hsa_dense_mask_bytes(0, 1, 1, 1) == 0
    one_row = lib.hsa_dense_mask_bytes(2, 1, 1, 300)            # 3 cells: 12 words a row, a byte a cell
    assert one_row == 256 + 256
    per_query = lib.hsa_dense_mask_bytes(1, 1, 200, 300)
    assert per_query >= 200 * 12 * 4 + 300 * 8 * 4 + 12 * 4 + 6
    assert lib.hsa_dense_mask_pack(P, 0, 0, 0, 1, 1, 1, 200, 300, P, per_query - 1, None) == -4
    assert lib.hsa_dense_mask_pack(None, 0, 0, 0, 1, 1, 1, 200, 300, P, per_query, None) == -1
    assert lib.hsa_dense_mask_pack(P, 0, 0, 0, 1, 1, 1, 200, 300, ctypes.c_void_p(0x1008), per_query, None) == -2


@pytest.mark.parametrize("bad", [dict(B=0), dict(H=3), dict(D=0), dict(D=300), dict(page=0), dict(pages=0), dict(width=0),
                                 dict(scale=0.0), dict(splits=0), dict(splits=1025), dict(algo=5), dict(table=None),
                                 dict(page=1 << 20, width=1 << 11)])
def test_paged_refuses(bad):
    assert paged(**bad) == -1


def test_paged_workspace():
    lib = _lib.load()
    assert paged(dtype=9) == -3
    need = lib.hsa_paged_attn_workspace_bytes(3, 4, 64, 5)
    assert need == 5 * 3 * 4 * 66 * 4
    assert paged(B=3, H=4, Hkv=4, splits=5) == -4
    assert paged(B=3, H=4, Hkv=4, splits=5, ws=P, nbytes=need - 1) == -4
    assert paged(B=3, H=4, Hkv=4, splits=5, ws=ctypes.c_void_p(0x1008), nbytes=need) == -2
    assert lib.hsa_paged_attn_workspace_bytes(3, 4, 64, 1) == 0


def test_split_choice():
    lib = _lib.load()
    assert lib.hsa_paged_attn_choose_splits(1, 8, 8, 16, 4) == 1          # 64 keys: one range
    assert 1 < lib.hsa_paged_attn_choose_splits(1, 8, 8, 64, 2048) <= 148
    assert lib.hsa_paged_attn_choose_splits(4096, 8, 8, 64, 2048) == 1
    assert lib.hsa_paged_attn_choose_splits(0, 8, 8, 64, 2048) == 1


def test_ops_refuse_cpu_tensors():
    q, k = torch.zeros(1, 3, 2, 8), torch.zeros(1, 5, 2, 8)
    with pytest.raises(_lib.HsaError):
        cross_attention(q, k, k)
    with pytest.raises(_lib.HsaError):
        paged_attention_decode(q[:, 0], k, k, torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32))
