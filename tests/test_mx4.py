"""MXFP4 without a GPU: the oracle pinned by literal values, shapes under FakeTensorMode, every refusal ahead of a
launch."""
import ctypes
import warnings

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from oracle import mx4_oracle as oracle
from sglite_amd import _lib, ops

NAN, INF = float("nan"), float("inf")


def block(*head):
    return torch.tensor(list(head) + [0.0] * (32 - len(head)), dtype=torch.float64)


def codes_of(x):
    c, s = oracle.quantize(x)
    return torch.stack((c & 15, c >> 4), -1).reshape(x.shape).tolist(), s.tolist()


def test_oracle_blocks():
    # A largest magnitude of 4 leaves the values as they are.
    c, s = codes_of(block(4, 0, 0.5, 1, 1.5, 2, 3, -4, -0.5, -3))
    assert s == [127] and c[:10] == [6, 0, 1, 2, 3, 4, 5, 14, 9, 13]
    # Ties go to the even code; beyond 6 to 6 (with a scale of 1 up to 8).
    c, s = codes_of(block(7.99, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 0.2500001, 0.7499, 5.0001, 6.9))
    assert s == [127] and c[:12] == [7, 0, 2, 2, 4, 4, 6, 6, 1, 1, 7, 7]
    assert codes_of(block(8, 1))[1] == [128] and codes_of(block(8, 1))[0][:2] == [6, 1]
    assert codes_of(block(3.999))[1] == [126] and codes_of(block(3.999))[0][0] == 7  # 7.998 -> 6
    # Zeros, the smallest scale, non-finite blocks; neighbours keep theirs.
    assert codes_of(block(0.0))[1] == [0]
    assert codes_of(block(2.0 ** -126))[1] == [0] and codes_of(block(2.0 ** -126))[0][0] == 4  # 2 * 2^-127
    assert codes_of(block(2.0 ** -130))[1] == [0] and codes_of(block(2.0 ** -130))[0][0] == 0
    assert codes_of(torch.cat((block(1, NAN), block(1), block(-INF))))[1] == [255, 125, 255]
    assert codes_of(block(2.0 ** 127))[1] == [252]


def test_oracle_values():
    codes = torch.tensor([[0x10, 0x32, 0x54, 0x76, 0x98, 0xBA, 0xDC, 0xFE] + [0] * 8], dtype=torch.uint8)
    v = oracle.values(codes, torch.tensor([[128]], dtype=torch.uint8))[0, :16]
    assert v.tolist() == [0, 1, 2, 3, 4, 6, 8, 12, 0, -1, -2, -3, -4, -6, -8, -12]
    assert oracle.values(codes, torch.tensor([[0]], dtype=torch.uint8))[0, 1] == 2.0 ** -128
    assert torch.isnan(oracle.values(codes, torch.tensor([[255]], dtype=torch.uint8))).all()


def test_oracle_keeps_what_it_made():
    x = torch.randn((7, 96), generator=torch.Generator().manual_seed(1)) * 10
    v = oracle.quantized(x)
    assert torch.equal(oracle.quantized(v), v)
    top = x.reshape(7, 3, 32).abs().amax(-1, keepdim=True).expand(7, 3, 32).reshape(7, 96)
    assert ((v - x).abs() <= top / 4).all()  # half a step of 2 (or 2 beyond 6) where the largest lies in [4, 8)


def test_weight_bytes():
    assert ops.mx4_weight_bytes(32, 128) == (2 * 1024, 2 * 256)
    assert ops.mx4_weight_bytes(8, 32) == (2 * 1024, 2 * 256)
    assert ops.mx4_weight_bytes(40, 544) == (4 * 5 * 1024, 4 * 2 * 256)
    for N, K in ((12, 32), (0, 32), (8, 0), (8, 48), (-8, 32)):
        with pytest.raises(ValueError):
            ops.mx4_weight_bytes(N, K)
    for N, K in ((8, 1 << 24), (1 << 24, 32)):
        with pytest.raises(RuntimeError):
            ops.mx4_weight_bytes(N, K)


def u8(*shape):
    return torch.zeros(shape, dtype=torch.uint8)


def test_block_refusals():
    for bad in (torch.zeros(4, 48), torch.zeros(()), torch.zeros(4, 0), torch.zeros(4, 32, dtype=torch.float64),
                torch.zeros(4, 32, dtype=torch.int32)):
        with pytest.raises(ValueError):
            ops.mx4_quantize(bad)
    with pytest.raises(ValueError, match="device tensors"):
        ops.mx4_quantize(torch.zeros(4, 32))
    for bad in (ops.Mx4(u8(4, 16), u8(4, 2)), ops.Mx4(u8(4, 16), u8(3, 1)), ops.Mx4(u8(4, 24), u8(4, 1)),
                ops.Mx4(u8(4, 16).char(), u8(4, 1)), ops.Mx4(u8(4, 16), u8(1)), ops.Mx4(u8(4, 16), u8(4, 1).int())):
        for call in (ops.mx4_dequantize, ops.mx4_repack):
            with pytest.raises(ValueError):
                call(bad)
    good = ops.Mx4(u8(8, 16), u8(8, 1))
    with pytest.raises(ValueError, match="float16"):
        ops.mx4_dequantize(good, torch.float64)
    for call in (ops.mx4_dequantize, ops.mx4_repack):
        with pytest.raises(ValueError, match="device tensors"):
            call(good)
    for bad in (ops.Mx4(u8(12, 16), u8(12, 1)), ops.Mx4(u8(16), u8(1)), ops.Mx4(u8(1, 1, 8, 16), u8(1, 1, 8, 1))):
        with pytest.raises(ValueError):
            ops.mx4_repack(bad)


def weight(N, K, E=None):
    wb, sb = ops.mx4_weight_bytes(N, K)
    return ops.Mx4Weight(u8(wb) if E is None else u8(E, wb), u8(sb) if E is None else u8(E, sb), N, K)


def test_gemm_refusals():
    x, w = torch.zeros(4, 64).half(), weight(64, 64)
    ok = dict(x=x, weight=w)
    for bad in (dict(x=x[0]), dict(x=x[:, :32]), dict(x=x.float()), dict(weight=w._replace(N=128)),
                dict(weight=w._replace(K=1024)), dict(weight=weight(64, 64, 2)), dict(weight=w._replace(w=w.w.char())),
                dict(weight=w._replace(w=u8(w.w.numel() + 1)[1:])), dict(activation="relu"),
                dict(weight=weight(32, 64), activation="silu")):
        with pytest.raises(ValueError):
            ops.mx4_gemm(**{**ok, **bad})
    for kw in ({}, dict(bias=torch.zeros(64)), dict(out=torch.zeros(4, 64).half())):
        with pytest.raises(ValueError, match="device tensors"):  # all else is in order
            ops.mx4_gemm(**ok, **kw)
    with pytest.raises(ValueError, match="one linear"):
        weight(64, 64).num_experts


def test_moe_refusals():
    i32 = torch.int32
    a, w, tw = torch.zeros(4, 64).half(), weight(64, 64, 3), torch.ones(4, 2)
    al = ops.MoeAlignment(torch.zeros(53, dtype=i32), torch.zeros(4, dtype=i32), torch.zeros(1, dtype=i32),
                          torch.zeros(4, dtype=i32))
    ok = dict(a=a, experts=w, align=al, topk_weights=tw, num_routed=8, top_k=2)
    for bad in (dict(experts=weight(64, 64)), dict(a=a[0]), dict(a=a[:, :32]), dict(a=a.float()), dict(activation="x"),
                dict(experts=weight(32, 64, 3), activation="gelu"), dict(topk_weights=None, mul_routed_weight=True),
                dict(topk_weights=tw[:3]), dict(num_routed=-1), dict(top_k=0),
                dict(align=al._replace(expert_offsets=torch.zeros(5, dtype=i32))),
                dict(align=al._replace(sorted_ids=torch.zeros(53, dtype=torch.int64)))):
        with pytest.raises(ValueError):
            ops.mx4_moe_gemm(**{**ok, **bad})
    with pytest.raises(ValueError, match="device tensors"):
        ops.mx4_moe_gemm(**ok)


INV, UNS, WSP = _lib.AWQ_STATUS_INVALID_ARGUMENT, _lib.AWQ_STATUS_UNSUPPORTED, _lib.AWQ_STATUS_WORKSPACE


def refused(want, status, kw):
    assert status == want, (kw, status)
    assert _lib.load().awq_last_error()


def test_c_abi_block_refusals():
    """Every bad call is turned away before a launch (the pointers are never read)."""
    lib = _lib.load()

    def call(x=4096, dtype=1, rows=4, K=64, codes=8192, scales=65, back=False):
        if back:
            return lib.awq_mx4_dequantize(codes, scales, rows, K, dtype, x, None)
        return lib.awq_mx4_quantize(x, dtype, rows, K, codes, scales, None)
    for back in (False, True):
        for want, kw in [(INV, dict(dtype=3)), (INV, dict(K=48)), (INV, dict(K=0)), (INV, dict(rows=-1)),
                         (INV, dict(x=None)), (INV, dict(codes=None)), (INV, dict(scales=None)), (INV, dict(x=4104)),
                         (INV, dict(codes=8194)), (UNS, dict(K=1 << 24)), (UNS, dict(rows=1 << 30, K=64))]:
            refused(want, call(back=back, **kw), kw)
        assert call(back=back, rows=0, x=None) == 0

    def pack(codes=4096, scales=65, E=2, N=64, K=64, w=8192, s=128, fn=lib.awq_mx4_repack):
        if fn is lib.awq_mx4_unrepack:
            return fn(w, s, E, N, K, codes, scales, None)
        return fn(codes, scales, E, N, K, w, s, None)
    for fn in (lib.awq_mx4_repack, lib.awq_mx4_unrepack):
        for want, kw in [(INV, dict(N=12)), (INV, dict(K=40)), (INV, dict(E=-1)), (INV, dict(E=1 << 17)),
                         (INV, dict(codes=None)), (INV, dict(scales=None)), (INV, dict(w=None)), (INV, dict(s=None)),
                         (INV, dict(codes=4100)), (INV, dict(w=8200)), (INV, dict(s=130)), (UNS, dict(N=1 << 24)),
                         (UNS, dict(E=65536, N=1 << 16))]:
            refused(want, pack(fn=fn, **kw), kw)
        assert pack(fn=fn, E=0, codes=None) == 0
    n = ctypes.c_int64()
    assert lib.awq_mx4_weight_bytes(64, 64, None, ctypes.byref(n)) == INV


def test_c_abi_product_refusals():
    lib = _lib.load()

    def gemm(x=4096, w=8192, s=128, bias=None, out=65536, M=4, N=64, K=64, dtype=0, act=0, ws=1 << 20, wsb=1 << 20):
        return lib.awq_mx4_gemm(x, w, s, bias, out, M, N, K, dtype, act, ws, wsb, None)
    big = dict(M=1 << 20, K=1 << 15)
    for want, kw in [(INV, dict(dtype=2)), (INV, dict(N=60)), (INV, dict(K=60)), (INV, dict(M=-1)), (INV, dict(act=3)),
                     (INV, dict(act=1, N=32)), (INV, dict(x=None)), (INV, dict(w=None)), (INV, dict(s=None)),
                     (INV, dict(out=None)), (INV, dict(x=4104)), (INV, dict(w=8200)), (INV, dict(s=130)),
                     (INV, dict(out=65544)), (INV, dict(bias=8)), (UNS, dict(K=1 << 24)), (UNS, dict(N=1 << 24)),
                     (UNS, dict(M=1 << 24)), (UNS, big), (WSP, dict(M=512, ws=None)), (WSP, dict(M=512, wsb=512)),
                     (WSP, dict(M=512, ws=(1 << 20) + 8))]:
        refused(want, gemm(**kw), kw)
    assert gemm(M=0, x=None, out=None) == 0
    assert lib.awq_mx4_workspace_bytes(0, 64, 64, 0) == 0 and lib.awq_mx4_workspace_bytes(-1, 64, 64, 0) == INV
    assert lib.awq_mx4_workspace_bytes(512, 64, 64, 0) >= 512 * (32 + 2)
    assert lib.awq_mx4_workspace_bytes(1, 64, 64, 5) == INV

    def moe(a=4096, rows=4, w=8192, s=128, E=3, N=64, K=64, dtype=0, ids=64, cap=100, off=128, tw=256, n=8, k=2, act=0,
            mul=1, out=65536, ws=1 << 20, wsb=1 << 20):
        return lib.awq_mx4_moe_gemm(a, rows, w, s, E, N, K, dtype, ids, cap, off, tw, n, k, act, mul, out, ws, wsb, None)
    for want, kw in [(INV, dict(dtype=2)), (INV, dict(N=60)), (INV, dict(K=60)), (INV, dict(act=3)),
                     (INV, dict(act=1, N=96)), (INV, dict(k=0)), (INV, dict(rows=3)), (INV, dict(a=None)),
                     (INV, dict(w=None)), (INV, dict(s=None)), (INV, dict(ids=None)), (INV, dict(off=None)),
                     (INV, dict(out=None)), (INV, dict(tw=None)), (INV, dict(a=4104)), (INV, dict(w=8194)),
                     (INV, dict(out=65544)), (UNS, dict(E=0)), (UNS, dict(E=513)), (UNS, dict(n=-1)),
                     (UNS, dict(n=1 << 24, rows=1 << 24)), (UNS, dict(cap=1 << 30)),
                     (UNS, dict(n=1 << 22, rows=1 << 22, k=1, K=256)), (WSP, dict(n=4096, rows=4096, ws=None))]:
        refused(want, moe(**kw), kw)
    assert moe(n=0, a=None, out=None) == 0 and moe(cap=0) == 0
    assert lib.awq_mx4_moe_workspace_bytes(0, 1, 3, 64, 64, 0) == 0
    assert lib.awq_mx4_moe_workspace_bytes(8, 0, 3, 64, 64, 0) == INV


def test_fake_shapes():
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")  # a fake tensor's address is 0, with a warning
        with FakeTensorMode():
            x = torch.empty((10, 96), dtype=torch.bfloat16, device="cuda")
            q = ops.mx4_quantize(x)
            assert q.codes.shape == (10, 48) and q.scales.shape == (10, 3) and q.codes.dtype == torch.uint8
            assert ops.mx4_dequantize(q, torch.float32).shape == (10, 96)
            w = ops.mx4_repack(ops.mx4_quantize(torch.empty((64, 96), device="cuda")))
            assert (w.w.numel(), w.s.numel()) == ops.mx4_weight_bytes(64, 96)
            assert ops.mx4_unrepack(w).codes.shape == (64, 48)
            assert ops.mx4_gemm(x, w).shape == (10, 64) and ops.mx4_gemm(x, w, activation="silu").shape == (10, 32)
            out = torch.empty((10, 64), dtype=torch.bfloat16, device="cuda")
            assert ops.mx4_gemm(x, w, out=out) is out
            ex = ops.mx4_repack(ops.mx4_quantize(torch.empty((4, 64, 96), device="cuda")))
            assert ex.num_experts == 4 and ex.expert(1).w.shape == w.w.shape
            align = ops.moe_align_block_size(torch.empty((10, 2), dtype=torch.int32, device="cuda"), 16, 4)
            assert ops.mx4_moe_gemm(x, ex, align, None, 20, 2, "gelu").shape == (20, 32)
