"""A 4-bit weight made an 8-bit one on the device: q4_dequant, then f8_pack. The codes are those of the dequantised values, and the product over them is within
the codes' half steps of the 4-bit weight's own."""
import numpy as np
import pytest

from oracle import f8
from oracle import oracle as O
from p0pc0rn_amd import capi
from tests.test_f8_gpu import Rows, activations

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("type_", ["f32", "f16"])
@pytest.mark.parametrize("M,N,K", [(1, 192, 288), (40, 1536, 2048)])
def test_from_a_packed_weight(dev, type_, M, N, K):
    rng = np.random.default_rng(N)
    packed, _ = O.pack_q4(O.randn(N * K, 5, 0.05), N, K)
    size, K8 = (4, 128 * f8.blocks(K)) if type_ == "f32" else (2, 128 * f8.blocks(K))
    q4, dense = capi.to_device(packed), capi.Buffer(size * N * K)
    w, ws = Rows(np.uint8, N, K8), Rows(np.float32, f8.blocks(N), K8 // 128)
    capi.q4_dequant(q4, N, K, **{"out32" if type_ == "f32" else "out16": dense})
    capi.f8_pack(capi.f8_pack_args(x=dense, type=capi.TYPE[type_], N=N, K=K, w=w.ptr, s=ws.ptr))
    values = dense.read(np.float32 if type_ == "f32" else np.float16, N * K).reshape(N, K).astype(np.float32)
    codes, scales = f8.pack(values)
    assert np.array_equal(w.read(), codes) and np.array_equal(ws.read(), scales)
    xc, xs = f8.quantise(activations(rng, M, K))
    x, s, y = Rows(np.uint8, M, K8, raw=xc), Rows(np.float32, K8 // 128, M, raw=xs), Rows(np.float32, M, N)
    capi.f8_gemm(capi.f8_gemm_args(x=x.ptr, xs=s.ptr, w=w.ptr, ws=ws.ptr, M=M, N=N, K=K8, type=0, y=y.ptr))
    a, v = f8.values(xc, xs)[:, :K], values.astype(np.float64)
    # a weight's code is within 2^-4 of it, or s 2^-10; sums in fp32 as in test_f8_gpu.py
    half = np.maximum(2.0 ** -4 * np.abs(v), np.repeat(np.repeat(scales, 128, 0)[:N], 128, 1)[:, :K].astype(np.float64) * 2.0 ** -10) * (1 + 2.0 ** -20)
    bound = np.abs(a) @ half.T + (128 + 2 * K8 / 128) * 2.0 ** -23 * (np.abs(a) @ (np.abs(v) + half).T)
    assert (np.abs(y.read() - a @ v.T) <= bound).all()
    for b in (q4, dense, w, ws, x, s, y):
        b.free()
