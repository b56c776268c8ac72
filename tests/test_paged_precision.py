"""Paged decode attention against its formula in 64 bits, within what the kernel's arithmetic leaves: scores and sums in fp32, q and
the weights as two values of the type each, one rounding of the output."""
import math

import pytest
import torch

from bitstack_b200 import _lib, glue

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(autouse=True)
def _status_is_clean():
    yield
    _lib.check_device_status()


def _requests(lens, hkv, ps, d, dtype, seed, wide):
    """Pages in random order, a table with `wide` spare columns; rows behind the last position hold NaN."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    held = [-(-n // ps) for n in lens]
    n = sum(held) + 2
    kp, vp = (torch.randn(n, hkv, ps, d, device=DEV, generator=g).to(dtype) for _ in range(2))
    order = torch.randperm(n, device=DEV, generator=g).int()
    table = torch.full((len(lens), max(max(held), 1) + wide), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, h in enumerate(held):
        table[b, :h] = order[at:at + h]
        at += h
        if lens[b] % ps:
            kp[int(table[b, h - 1]), :, lens[b] % ps:] = vp[int(table[b, h - 1]), :, lens[b] % ps:] = float("nan")
    kp[order[at:].long()] = vp[order[at:].long()] = float("nan")
    return kp, vp, table, g


def _rows(pages, table, b, n, ps):
    """[kv heads, n, d] of request b; writes go to the pages through `_put`."""
    return pages[table[b, :-(-n // ps)].long()].transpose(0, 1).reshape(pages.shape[1], -1, pages.shape[3])[:, :n]


def _put(pages, table, b, n, ps, rows):
    """rows [kv heads, n, d] into the pages of request b."""
    p = torch.arange(n, device=DEV)
    pages[table[b, p // ps].long(), :, p % ps] = rows.transpose(0, 1)


def _plain_rotary(n, d, dtype):
    return torch.ones(n, d, device=DEV, dtype=dtype), torch.zeros(n, d, device=DEV, dtype=dtype)


def _check(out, q, cos, sin, lens, table, kp, vp, hq, hkv, d, ps, dtype):
    """kp, vp: the pages after the call, so the new key is the rounded one.  In units of the weights, relative:
    a score: q as two values 'half^2', below the type's normal range 2^-25 of fp16 absolutely; rotation, products and sums in fp32 (d + 5)
      2^-24 of sum |q||k| / sqrt(d).  A change of all scores by that much moves a weight by twice as much (its own and the sum's);
    a weight: as two values 'half^2'; exponential and its argument 2^-17 for weights that count (two roundings of an argument of at most
      64, 2^-22 of the approximation); fp32 sums 2^-16 (at most 128 steps of a chain, 2^-23 each).
    fp16 weights below their normal range: 2^-25 at a scale of 2^13 for the largest weight, hence 2^-38 of the sum of all |v|.
    One rounding of the output, half a step (2^-25 below fp16's normal range)."""
    half = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    worst = 0.0
    for b, n in enumerate(lens):
        if n == 0:
            assert bool((out[b] == 0).all())
            continue
        x = q[b].reshape(hq, d).double()
        c, s = cos[n - 1].double(), sin[n - 1].double()
        other = torch.cat([-x[:, d // 2:], x[:, :d // 2]], -1)
        qr, qa = (x * c + other * s).view(hkv, -1, d), ((x * c).abs() + (other * s).abs()).view(hkv, -1, d)
        keys, values = _rows(kp, table, b, n, ps).double(), _rows(vp, table, b, n, ps).double()
        p = torch.softmax(qr @ keys.transpose(1, 2) / math.sqrt(d), -1)
        ref = p @ values
        size = ((qa * (half * half + (d + 5) * 2.0 ** -24) + tiny) @ keys.abs().transpose(1, 2) / math.sqrt(d)).amax(-1, keepdim=True)
        tol = (2 * size + half * half + 2.0 ** -17 + 2.0 ** -16) * (p @ values.abs()) + half * ref.abs() + 2.0 ** -24
        if dtype == torch.float16:
            tol = tol + 2.0 ** -38 * values.abs().sum(1, keepdim=True)
        err = (out[b].view(hkv, -1, d).double() - ref).abs()
        assert bool(torch.isfinite(out[b]).all()), b
        worst = max(worst, float((err / tol).max()))
    assert worst <= 1, worst


_FORMS = [  # query heads, kv heads, head_dim, page size: every form of the kernel (up to 8 / more heads, pages of 16 rows or not)
    (8, 2, 128, 16), (8, 2, 128, 24), (4, 1, 64, 16), (4, 1, 64, 7), (20, 1, 128, 32), (20, 1, 128, 24), (24, 2, 64, 64), (33, 1, 64, 9), (9, 1, 128, 1)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv,d,ps", _FORMS)
def test_random_requests(hq, hkv, d, ps, dtype):
    """(The bound sees a lost stretch of 16 positions at all of these lengths, bf16 among them: checked on the exact weights.)"""
    for lens, wide in (([500, 1, 0, 129, 64, 17], 0), ([1100, 63, 2049, 0, 1, 300], 40)):   # one CTA per pair; shared by CTAs
        kp, vp, table, g = _requests(lens, hkv, ps, d, dtype, hq * 100 + ps, wide * 128 // ps)
        q, k, v = (torch.randn(len(lens), h * d, device=DEV, generator=g).to(dtype) for h in (hq, hkv, hkv))
        a = torch.outer(torch.arange(max(lens), device=DEV, dtype=torch.float64), 1.0 / 10000.0 ** (torch.arange(0, d, 2, device=DEV, dtype=torch.float64) / d))
        cos, sin = (torch.cat([t, t], -1).to(dtype) for t in (a.cos(), a.sin()))
        out = glue.paged_decode_attention(q, k, v, cos, sin, torch.tensor([n - 1 for n in lens], device=DEV), table, kp, vp, hq, hkv, d)
        _check(out, q, cos, sin, lens, table, kp, vp, hq, hkv, d, ps, dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv,d,ps", _FORMS)
def test_every_stretch_of_positions_counts_once(hq, hkv, d, ps, dtype):
    """Equal keys, and values that mark their stretch of 16 positions in a dimension of their own (every d-th shares one): a stretch
    that is left out, taken twice or taken for another one shows in its dimension."""
    half = torch.finfo(dtype).eps / 2
    for lens, wide in (([512, 1, 0, 129, 64, 17, 255], 0), ([2049, 33, 0, 700, 1, 3000, 65, 1999, 128, 16], 60), ([40000], 0)):
        kp, vp, table, _ = _requests(lens, hkv, ps, d, dtype, hq + ps, wide * 128 // ps)
        v = torch.zeros(len(lens), hkv * d, device=DEV, dtype=dtype)
        for b, n in enumerate(lens):
            if n:
                mark = torch.nn.functional.one_hot(torch.arange(n, device=DEV) // 16 % d, d).to(dtype)
                _put(kp, table, b, n, ps, torch.zeros(hkv, n, d, device=DEV, dtype=dtype))
                _put(vp, table, b, n, ps, mark.expand(hkv, n, d))
                v[b] = mark[n - 1].repeat(hkv)
        q, k = torch.randn(len(lens), hq * d, device=DEV, dtype=dtype), torch.zeros(len(lens), hkv * d, device=DEV, dtype=dtype)
        cos, sin = _plain_rotary(max(lens), d, dtype)
        out = glue.paged_decode_attention(q, k, v, cos, sin, torch.tensor([n - 1 for n in lens], device=DEV), table, kp, vp, hq, hkv, d)
        for b, n in enumerate(lens):
            want = torch.zeros(d, dtype=torch.float64, device=DEV)
            if n:
                want = torch.bincount(torch.arange(n, device=DEV) // 16 % d, minlength=d).double() / n
            err = (out[b].view(hq, d).double() - want).abs()
            # all weights are equal and exact: fp32 sums, one rounding
            assert bool((err <= (half + 2.0 ** -16) * want + 2.0 ** -25).all()), (b, n)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,lead,hkv", [(400, 14.0, 1), (500, 18.0, 8), (4096, 18.0, 1), (60001, 16.0, 1), (131071, 17.5, 1), (131071, 21.0, 1),
                                        (8193, 12.0, 64), (8193, 17.5, 64), (8193, 20.0, 64)])
def test_many_small_weights_beside_a_large_one(n, lead, hkv, dtype):
    """One key leads by `lead` (in nats).  What the other positions give together is as exact as the rest, whether the leading
    value is zero (all of the output is theirs) or one (they bring it to one).  64 kv heads: a warp keeps over 1000 positions."""
    hq, d, ps = 4 if hkv == 1 else hkv, 64, 16
    kp, vp, table, g = _requests([n] * 4, hkv, ps, d, dtype, 3, 0)
    q = torch.zeros(4, hq, d, device=DEV, dtype=dtype)
    q[:, :, 0] = lead                                  # lead * 8 / sqrt(64)
    q[:, hq // 2:, 1] = 0.5                            # heads whose other weights spread a little
    for b in range(4):
        keys = torch.zeros(hkv, n, d, device=DEV, dtype=dtype)
        keys[:, :, 1] = torch.randn(n, device=DEV, generator=g).to(dtype)
        values = torch.ones(hkv, n, d, device=DEV, dtype=dtype)
        values[:, :, d // 2:] = torch.rand(n, d // 2, device=DEV, generator=g).to(dtype)
        at = (0, n // 2, n // 3, 1)[b]                 # a first position as sink, and others
        keys[:, at] = 0
        keys[:, at, 0] = 8.0
        if b < 2:
            values[:, at] = 0
        _put(kp, table, b, n, ps, keys)
        _put(vp, table, b, n, ps, values)
    cos, sin = _plain_rotary(n, d, dtype)
    k, v = torch.zeros(4, hkv * d, device=DEV, dtype=dtype), torch.ones(4, hkv * d, device=DEV, dtype=dtype)
    q = q.view(4, hq * d)
    out = glue.paged_decode_attention(q, k, v, cos, sin, torch.full((4,), n - 1, device=DEV), table, kp, vp, hq, hkv, d)
    _check(out, q, cos, sin, [n] * 4, table, kp, vp, hq, hkv, d, ps, dtype)


@pytest.mark.parametrize("dtype,most", [(torch.float16, 3.0e4), (torch.bfloat16, 1.0e8)])
@pytest.mark.parametrize("n", [300, 1500])
def test_scores_far_beyond_one(n, dtype, most):
    """Finite q and keys whose scores are in the thousands of millions: the two equal largest ones share everything."""
    hq, hkv, d, ps = 6, 2, 128, 16
    kp, vp, table, g = _requests([n], hkv, ps, d, dtype, n, 0)
    level = torch.rand(n, device=DEV, generator=g) * 0.5 + 0.25       # of the largest: far enough below it
    level[5] = level[n - 100] = 1.0
    keys = (level * most)[None, :, None].expand(hkv, n, d).to(dtype)
    _put(kp, table, 0, n, ps, keys)
    q = (most * torch.tensor([1.0, 0.93, 0.77, 0.61, 0.53, 0.37], device=DEV))[:, None].expand(hq, d).to(dtype).reshape(1, hq * d).contiguous()
    cos, sin = _plain_rotary(n, d, dtype)
    v = torch.randn(1, hkv * d, device=DEV, generator=g).to(dtype)
    out = glue.paged_decode_attention(q, keys[:, n - 1].reshape(1, hkv * d), v, cos, sin, torch.tensor([n - 1], device=DEV), table, kp, vp, hq, hkv, d)
    values = _rows(vp, table, 0, n, ps).double()
    want = ((values[:, 5] + values[:, n - 100]) / 2).repeat_interleave(hq // hkv, 0)
    err = (out.view(hq, d).double() - want).abs()
    assert bool((err <= (torch.finfo(dtype).eps / 2 + 2.0 ** -16) * want.abs() + 2.0 ** -24).all()), float(err.max())   # (NaN fails)
