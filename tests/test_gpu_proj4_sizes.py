"""GPU: 4-bit projections at the ends of what their scales may be."""
import numpy as np
import pytest
import torch

from bitgpu_amd import engine as E
from tests.linear_helpers import cuda
from tests.test_gpu_proj4 import Weight, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M", [1, 3, 6, 16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("mins", [False, True])
@pytest.mark.parametrize("power", [-100, 90])
def test_scales(dev, M, group, mins, power):
    """Scales up to 2^90 (and far below one) where all values and codes of a group are as large as they get."""
    rng = np.random.default_rng(M + group)
    w = Weight(rng, 64, 640, group, mins, f16=False)
    w.scale[:] = 2.0 ** power
    w.scale[::3, ::2] *= 0.75
    if mins:
        w.min[:] = -w.scale * 7
    w.code[:16] = 15
    w.code[16:32] = 0
    words = np.zeros_like(w.words)
    for i in range(8):
        words |= w.code[:, i::8].astype(np.uint32) << np.uint32(4 * i)
    w.words = words
    x = rng.standard_normal((M, 640)).astype(np.float32)
    x[M - 1] = 1.999999
    out = torch.empty(M, 64, device="cuda")
    E.fused_mm(w.handle(), cuda(x), [out])
    got = out.cpu().numpy()
    assert np.isfinite(got).all()
    check(got, w, x)
