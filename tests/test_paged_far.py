"""Serving operators where offsets pass 32 bits: pages far into a large pool, rows of logits far apart."""
import pytest
import torch

from bitstack_b200 import _lib, glue
from test_paged_precision import _check
from test_paged_serving import _check_sample

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(autouse=True)
def _status_is_clean():
    yield
    _lib.check_device_status()


def test_pages_far_into_the_pool():
    """A pool of 2^31 + elements for K and V side by side; the requests' pages are the last ones and the first."""
    hq, hkv, d, ps, dtype = 8, 2, 128, 512, torch.float16
    pages = 2 ** 31 // (2 * hkv * ps * d) + 8
    both = torch.empty(pages, 2, hkv, ps, d, device=DEV, dtype=dtype)
    kp, vp = both[:, 0], both[:, 1]
    assert (pages - 1) * kp.stride(0) > 2 ** 31
    g = torch.Generator(device=DEV).manual_seed(1)
    table = torch.tensor([[pages - 1, 0, pages - 2], [pages - 3, pages - 4, -1]], dtype=torch.int32, device=DEV)
    for p in table[table >= 0].tolist():
        both[p] = torch.randn(2, hkv, ps, d, device=DEV, generator=g).to(dtype)
    a = torch.outer(torch.arange(1500, device=DEV, dtype=torch.float64), 1.0 / 10000.0 ** (torch.arange(0, d, 2, device=DEV, dtype=torch.float64) / d))
    cos, sin = (torch.cat([t, t], -1).to(dtype) for t in (a.cos(), a.sin()))
    # a prompt's last 600 tokens of request 0 through the rotary write, then one step of both requests
    T, lens = 600, [1401, 1000]
    q, k, v = (torch.randn(T, h * d, device=DEV, generator=g).to(dtype) for h in (hq, hkv, hkv))
    pos = torch.arange(lens[0] - 1 - T, lens[0] - 1, device=DEV)
    slots = table[0][pos // ps].long() * ps + pos % ps
    glue.rope_paged_cache(q, k, v, cos, sin, pos, slots, kp, vp, hq, hkv, d)
    assert torch.equal(vp[table[0][pos // ps].long(), :, pos % ps], v.view(T, hkv, d))
    c, s = cos[pos].double()[:, None], sin[pos].double()[:, None]
    x = k.view(T, hkv, d).double()
    ref = x * c + torch.cat([-x[..., d // 2:], x[..., :d // 2]], -1) * s
    err = (kp[table[0][pos // ps].long(), :, pos % ps].double() - ref).abs()
    assert bool((err <= 2.0 ** -11 * ref.abs() + 3 * 2.0 ** -24 * 2 * x.abs().amax() + 2.0 ** -24).all())   # one rounding, fp32 products
    q, k, v = (torch.randn(2, h * d, device=DEV, generator=g).to(dtype) for h in (hq, hkv, hkv))
    out = glue.paged_decode_attention(q, k, v, cos, sin, torch.tensor([n - 1 for n in lens], device=DEV), table, kp, vp, hq, hkv, d)
    _check(out, q, cos, sin, lens, table, kp, vp, hq, hkv, d, ps, dtype)


def test_rows_of_logits_far_apart():
    V, stride = 5000, 2 ** 31 + 8
    big = torch.empty(stride + V, device=DEV, dtype=torch.float16)
    logits = big.as_strided((2, V), (stride, 1))
    logits.copy_(torch.randn(2, V, device=DEV, generator=torch.Generator(device=DEV).manual_seed(2)) * 3)
    _check_sample(logits, torch.tensor([0.3, 0.8], device=DEV), top_p=[0.9, 0.95])
