"""Sampling from rows whose tokens are (nearly) all alike: the sums of the weights are as large as they can get."""
import pytest
import torch

from bitstack_b200 import _lib
from test_paged_serving import _check_sample

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(autouse=True)
def _status_is_clean():
    yield
    _lib.check_device_status()


@pytest.mark.parametrize("V", [4097, 8192, 8193, 16384, 24759, 32000, 50257, 93510, 128256, 238855, 262144])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_flat_rows(V, dtype):
    g = torch.Generator(device=DEV).manual_seed(V)
    rows = torch.stack([torch.full((V,), -7.0, device=DEV), torch.randn(V, device=DEV, generator=g) * 1e-3,
                        -(torch.arange(V, device=DEV) % 61) * 1e-3, torch.randn(V, device=DEV, generator=g) * 3])
    logits, u = rows.to(dtype), torch.tensor([0.5, 0.422103, 0.999, 0.932773], device=DEV)
    _check_sample(logits, u)
    _check_sample(logits, u, temperature=[1.0, 0.7, 1.3, 100.0])
    _check_sample(logits, u, temperature=[1.0, 1.0, 30.0, 100.0], top_p=[0.9, 0.5, 0.95, 0.999])
    _check_sample(logits, u, temperature=[1.0, 1.0, 1.0, 100.0], top_k=[V // 2 + 1, V - 1, 1000, V // 3], top_p=[1.0, 0.9, 0.3, 0.7])
    _check_sample(logits, u, temperature=[100.0] * 4, min_p=[0.1, 0.5, 0.98, 1e-9], top_p=[1e-3, 1.0, 0.1, 1.0])
