"""Calls that fill all blocks of their kernels: normalisation of many fp32 rows and of rows of single numbers, routing of many tokens of 512 experts.  The bounds are
those of the operators' own tests."""
import pytest
import torch

import test_balanced_router
import test_layer_norm

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("rows,H,dtype", [(3000, 4096, F32), (2500, 2049, F32), (2500, 2049, BF), (1500, 7169, F32), (1200, 8191, BF), (700, 12288, BF), (600, 16384, F32)])
def test_normalisation(native, rows, H, dtype):
    for center in (True, False):
        t, dy, dsum = test_layer_norm.make(rows, H, dtype, F32, seed=H, bias=center)
        test_layer_norm.check(t, center, dy, dsum)


@pytest.mark.parametrize("T,E", [(20000, 512), (9600, 300)])
def test_routing(native, T, E):
    test_balanced_router.check(T, 512, E, 8, 4, seed=E)
    test_balanced_router.check(T, 136, E, 3, 1, renormalize=False, masked=0.3, seed=E)
