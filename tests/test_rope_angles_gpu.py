"""The rotation's cosines and sines themselves: heads whose pairs are (1, 0), of which fp32 results hold them as they are.

Bound: a cosine is rounded by the function that makes it and by the sum that turns it on, each by up to 2^-25 (half a step below 1) and so by 2^-25 / sqrt 3 in the
mean square; two such are 2.43e-8. The frequency, 10 roundings of 2^-53 at positions below 2^20, adds 1.2e-9 at most. An angle that goes on in 32 bits is off by up to
2 pi 2^-26 by itself, 3.2e-8 with the rest in the mean square."""
import numpy as np
import pytest

from p0pc0rn_amd import capi

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mode", ["inter", "half"])
@pytest.mark.parametrize("far", [300, 1 << 17, 1 << 20])
def test_cosines_and_sines(dev, mode, far):
    rows, dim = 4096, 128
    pos = np.random.default_rng(far).integers(0, far, rows).astype(np.int32)
    pos[0] = 0
    x = np.zeros((rows, dim), np.float32)
    first = np.s_[:, 0::2] if mode == "inter" else np.s_[:, :dim // 2]
    second = np.s_[:, 1::2] if mode == "inter" else np.s_[:, dim // 2:]
    x[first] = 1
    xb, yb, pb = capi.to_device(x), capi.Buffer(x.nbytes), capi.to_device(pos)
    capi.rope(capi.rope_args(x=xb, y=yb, type=0, rows=rows, hq=1, dim=dim, mode=capi.ROPE[mode], pos=pb))
    got = yb.read(np.float32, x.size).reshape(rows, dim).astype(np.float64)
    angle = pos[:, None].astype(np.longdouble) * np.longdouble(10000) ** -(np.arange(dim // 2, dtype=np.longdouble) / (dim // 2))
    err = np.concatenate([got[first] - np.cos(angle), got[second] - np.sin(angle)]).astype(np.float64)
    assert np.sqrt((err ** 2).mean()) <= 2.43e-8 + 1.2e-9
    assert (got[first][0] == 1).all() and (got[second][0] == 0).all()
    for b in (xb, yb, pb):
        b.free()
