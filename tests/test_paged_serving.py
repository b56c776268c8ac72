"""The serving operators on the GPU against plain implementations in 64 bits: page bookkeeping, rotary cache writes, paged
decode attention, sampling."""
import math
from fractions import Fraction

import numpy as np
import pytest
import torch

from bitstack_b200 import _lib, glue

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(autouse=True)
def _status_is_clean():
    yield
    _lib.check_device_status()


def _gen(*key):
    return torch.Generator(device=DEV).manual_seed(hash(key) % (1 << 31) if not all(isinstance(k, int) for k in key) else sum(k * 7919 ** i for i, k in enumerate(key)) % (1 << 31))


def _half_step(t):
    return torch.finfo(t).eps / 2


# ------------------------------------------------------------------------------------------------ page bookkeeping

def _ref_tables(lens, new, table, free, count, ps, max_tokens):
    lens, new, table = lens.tolist(), new.tolist(), table.clone()
    width, need_before, taken = table.shape[1], 0, 0
    slots, positions, offsets, last, out = [], [], [0], [], []
    for b, (n, add) in enumerate(zip(lens, new)):
        add = max(add, 0)
        held, after = -(-n // ps), -(-(n + add) // ps)
        fits = after <= width
        need = after - held if fits else 0
        served = fits and (need == 0 or need_before + need <= count)
        if served:
            for j in range(need):
                table[b, held + j] = free[count - 1 - need_before - j]
            taken += need
        for p in range(n, n + add):
            positions.append(p if served else -1)
            slots.append(int(table[b, p // ps]) * ps + p % ps if served else -1)
        need_before += need
        offsets.append(offsets[-1] + add)
        last.append(n + add - 1 if served and add else -1)
        out.append(n + add if served else n)
    pad = [-1] * max_tokens
    return table, (slots + pad)[:max_tokens], (positions + pad)[:max_tokens], offsets, last, out, count - taken


@pytest.mark.parametrize("batch,ps,most,grow,short,width", [
    (1, 16, 1, 1, 0, 4), (5, 1, 9, 1, 0, 40), (33, 16, 100, 1, 0, 12), (40, 24, 300, 200, 0, 40), (40, 24, 300, 200, 9, 40),
    (64, 8, 100, 60, 30, 16), (1500, 16, 70, 1, 11, 8), (2100, 4, 20, 9, 0, 16),
    (5120, 16, 20, 1, 0, 3), (6144, 16, 20, 1, 5, 3), (8192, 16, 20, 1, 0, 3)])
def test_page_tables(batch, ps, most, grow, short, width):
    g = torch.Generator().manual_seed(batch * 31 + ps)
    lens = torch.randint(0, most + 1, (batch,), generator=g, dtype=torch.int32)
    lens[0] = 0
    new = torch.randint(0, grow + 1, (batch,), generator=g, dtype=torch.int32)
    if batch > 4:
        new[3] = -5                                   # counts as none
    if batch > 30:
        lens[7], new[7] = width * ps, 1               # its row is full
    held = (lens + ps - 1) // ps
    need = int(((lens + new.clamp(min=0) + ps - 1) // ps - held).sum())
    pool = torch.randperm(int(held.sum()) + need + 5, generator=g).int()
    table = torch.full((batch, width), -7, dtype=torch.int32)
    at = 0
    for b in range(batch):
        n = int(held[b])
        table[b, :n] = pool[at:at + n]
        at += n
    free = torch.full((need + 20,), -9, dtype=torch.int32)
    count = max(need - short, 0)
    free[:count] = pool[at:at + count]
    tokens = int(new.clamp(min=0).sum()) + 3
    want = _ref_tables(lens, new, table, free, count, ps, tokens)
    d = [t.to(DEV) for t in (lens, new, table, free, torch.tensor([count], dtype=torch.int32))]
    for in_place in (False, True):
        lo, co, tab = torch.empty_like(d[0]), torch.empty_like(d[4]), d[2].clone()
        wide = torch.full((batch, width + 5), -3, dtype=torch.int32, device=DEV)   # a view with a row stride of its own
        wide[:, :width] = tab
        kw = {} if in_place else dict(lens_out=lo, free_count_out=co)
        slots, positions, offsets, last = glue.page_tables(d[0], d[1], wide[:, :width], d[3], d[4], ps, tokens, **kw)
        if in_place:
            lo, co = d[0], d[4]
        assert torch.equal(wide[:, :width].cpu(), want[0]) and bool((wide[:, width:] == -3).all())
        for got, ref in zip((slots, positions, offsets, last, lo), want[1:6]):
            assert got.tolist() == ref
        assert int(co) == want[6]
    assert torch.equal(d[3].cpu(), free)              # the stack's entries stay


def test_page_tables_without_a_list_and_with_a_short_one():
    lens, new = torch.tensor([3, 16, 0], dtype=torch.int32, device=DEV), torch.tensor([1, 1, 2], dtype=torch.int32, device=DEV)
    table = torch.tensor([[4, -1], [2, -1], [-1, -1]], dtype=torch.int32, device=DEV)
    free, count = torch.tensor([9, 8, 7], dtype=torch.int32, device=DEV), torch.tensor([3], dtype=torch.int32, device=DEV)
    slots, positions, offsets, last = glue.page_tables(lens, new, table, free, count, 16)
    assert slots.numel() == 0 and offsets.tolist() == [0, 1, 2, 4] and last.tolist() == [3, 16, 1] and lens.tolist() == [4, 17, 2]
    assert table.tolist() == [[4, -1], [2, 7], [8, -1]] and count.tolist() == [1]
    slots, positions, _, _ = glue.page_tables(lens, new, table, free, count, 16, max_tokens=2)
    assert slots.tolist() == [4 * 16 + 4, 7 * 16 + 1] and positions.tolist() == [4, 17]
    with pytest.raises(_lib.BitStackDeviceIndexError):
        _lib.check_device_status()


def test_release_then_reuse_in_order():
    ps, R, P = 8, 6, 5
    lens = torch.tensor([17, 0, 8, 40, 1, 9], dtype=torch.int32, device=DEV)
    held = [3, 0, 1, 5, 1, 2]
    table = torch.full((R, P), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(held):
        table[b, :n] = torch.arange(at, at + n)
        at += n
    free, count = torch.full((at + 2,), -1, dtype=torch.int32, device=DEV), torch.tensor([2], dtype=torch.int32, device=DEV)
    free[0], free[1] = at, at + 1
    done = torch.tensor([True, True, False, True, False, False], device=DEV)
    glue.release_pages(done, lens, table, free, count, ps)
    assert lens.tolist() == [0, 0, 8, 0, 1, 9] and count.tolist() == [10]
    assert free[:10].tolist() == [at, at + 1, 0, 1, 2, 4, 5, 6, 7, 8]
    new = torch.tensor([0, 9, 1, 0, 0, 0], dtype=torch.int32, device=DEV)
    glue.page_tables(lens, new, table, free, count, ps)
    assert table[1, :2].tolist() == [8, 7] and table[2, :2].tolist() == [3, 6] and count.tolist() == [7]
    free2, full = torch.zeros(1, dtype=torch.int32, device=DEV), torch.tensor([1], dtype=torch.int32, device=DEV)
    glue.release_pages(torch.ones(R, dtype=torch.bool, device=DEV), lens, table, free2, full, ps)   # no room: reported, not written
    assert full.tolist() == [1]
    with pytest.raises(_lib.BitStackDeviceIndexError):
        _lib.check_device_status()


# ------------------------------------------------------------------------------------------------ rotary write and attention

def _tables_of_rotary(n, dim, dtype):
    a = torch.outer(torch.arange(n, dtype=torch.float64), 1.0 / (10000.0 ** (torch.arange(0, dim, 2, dtype=torch.float64) / dim)))
    a = torch.cat([a, a], -1)
    return a.cos().to(dtype).to(DEV), a.sin().to(dtype).to(DEV)


def _turn(x, cos, sin):
    """x [T, heads, D] float64; (rotated, sum of the magnitudes of its two products)."""
    h = x.shape[-1] // 2
    other = torch.cat([-x[..., h:], x[..., :h]], -1)
    return x * cos[:, None] + other * sin[:, None], (x * cos[:, None]).abs() + (other * sin[:, None]).abs()


def _pool(n, hkv, ps, d, dtype, g, interleaved):
    if interleaved:                                    # K and V of a page side by side in one allocation
        both = torch.randn(n, 2, hkv, ps, d, device=DEV, generator=g).to(dtype)
        return both[:, 0], both[:, 1]
    return torch.randn(n, hkv, ps, d, device=DEV, generator=g).to(dtype), torch.randn(n, hkv, ps, d, device=DEV, generator=g).to(dtype)


def _qkv_rows(T, hq, hkv, d, dtype, g, fused):
    if fused:                                          # views of one projection output
        x = torch.randn(T, (hq + 2 * hkv) * d + 8, device=DEV, generator=g).to(dtype)
        return x[:, :hq * d], x[:, hq * d:(hq + hkv) * d], x[:, (hq + hkv) * d:(hq + 2 * hkv) * d]
    return tuple(torch.randn(T, h * d, device=DEV, generator=g).to(dtype) for h in (hq, hkv, hkv))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,hq,hkv,d,ps,fused", [(1, 4, 2, 128, 16, False), (37, 8, 2, 64, 24, True), (130, 3, 3, 128, 1, False),
                                                 (9, 32, 8, 128, 64, True), (5, 2, 1, 80, 8, False), (3, 1, 1, 16, 5, False)])
def test_rope_paged_cache(T, hq, hkv, d, ps, fused, dtype):
    g = _gen(T, hq, d, ps)
    q, k, v = _qkv_rows(T, hq, hkv, d, dtype, g, fused)
    cos, sin = _tables_of_rotary(200, d, dtype)
    n = -(-T // ps) + 4
    kp, vp = _pool(n, hkv, ps, d, dtype, g, fused)
    pos = torch.randint(0, 200, (T,), device=DEV, generator=g)
    slots = torch.randperm(n * ps, device=DEV, generator=g)[:T].clone()
    if T > 4:
        pos[T - 2:], slots[T - 2:] = -1, -1            # padding
        slots[0] = -1                                  # turned, not cached
        pos[1] = -1                                    # padding with a slot: nothing is cached
    q0, k0, kp0, vp0 = q.clone(), k.clone(), kp.clone(), vp.clone()
    out = glue.rope_paged_cache(q, k, v, cos, sin, pos, slots, kp, vp, hq, hkv, d)
    assert torch.equal(q, q0) and torch.equal(k, k0)
    at = pos.clamp(min=0)
    c, s = cos[at].double(), sin[at].double()
    # one rounding to the type, and three fp32 roundings of the two products
    for got, x, heads in ((out, q, hq), (None, k, hkv)):
        ref, size = _turn(x.reshape(T, heads, d).double(), c, s)
        if got is not None:
            ref[pos < 0], size[pos < 0] = 0, 0
            err = (got.view(T, heads, d).double() - ref).abs()
            assert bool((err <= _half_step(dtype) * ref.abs() + 3 * 2 ** -24 * size + 1e-7 * (size > 0)).all())
        else:
            k_ref, k_size = ref, size
    touched = torch.zeros(n * ps, dtype=torch.bool, device=DEV)
    for t in range(T):
        if int(slots[t]) < 0 or int(pos[t]) < 0:
            continue
        page, row = int(slots[t]) // ps, int(slots[t]) % ps
        touched[int(slots[t])] = True
        err = (kp[page, :, row].double() - k_ref[t]).abs()
        assert bool((err <= _half_step(dtype) * k_ref[t].abs() + 3 * 2 ** -24 * k_size[t] + 1e-7).all())
        assert torch.equal(vp[page, :, row], v[t].reshape(hkv, d))
    keep = ~touched.view(n, ps)
    assert torch.equal(kp.transpose(1, 2)[keep], kp0.transpose(1, 2)[keep]) and torch.equal(vp.transpose(1, 2)[keep], vp0.transpose(1, 2)[keep])


def test_rope_paged_cache_does_not_follow_bad_indices():
    g = _gen(1, 2, 3)
    q, k, v = _qkv_rows(4, 2, 1, 64, torch.float16, g, False)
    cos, sin = _tables_of_rotary(10, 64, torch.float16)
    kp, vp = _pool(3, 1, 4, 64, torch.float16, g, False)
    k0, v0 = kp.clone(), vp.clone()
    out = glue.rope_paged_cache(q, k, v, cos, sin, torch.tensor([3, 10, 4, 5], device=DEV), torch.tensor([12, 1, -4, 1 << 40], device=DEV), kp, vp, 2, 1, 64)
    assert torch.equal(kp, k0) and torch.equal(vp, v0)
    assert torch.isnan(out[1]).all() and torch.isfinite(out[[0, 2, 3]]).all()
    with pytest.raises(_lib.BitStackDeviceIndexError):
        _lib.check_device_status()


def _make_requests(lens, hkv, ps, d, dtype, g, interleaved=False, poison=True):
    held = [-(-n // ps) for n in lens]
    n = sum(held) + 3
    kp, vp = _pool(n, hkv, ps, d, dtype, g, interleaved)
    order = torch.randperm(n, device=DEV, generator=g).int()
    table = torch.full((len(lens), max(max(held), 1) + 2), -1, dtype=torch.int32, device=DEV)   # entries behind a request's pages: never read
    at = 0
    for b, h in enumerate(held):
        table[b, :h] = order[at:at + h]
        at += h
    if poison:                                         # rows behind the last position hold garbage
        for b, m in enumerate(lens):
            if m % ps:
                page = int(table[b, (m - 1) // ps])
                kp[page, :, m % ps:], vp[page, :, m % ps:] = float("nan"), float("inf")
        spare = order[at:].long()
        kp[spare], vp[spare] = float("nan"), float("nan")
    return kp, vp, table


def _check_attention(out, q, k, v, cos, sin, lens, table, kp, vp, hq, hkv, d, ps, dtype):
    """kp, vp: the pages after the call.  Rounding q to the type moves a score by at most half a step of sum |q||k| / sqrt(D),
    fp32 accumulation by (D + 2) 2^-24 of it; a weight moves by twice the largest such change, by half a step where the weights
    are rounded to the type for the product, and 2^-18 covers exp and fp32 sums; then one rounding of the output."""
    B, half = len(lens), _half_step(dtype)
    for b, n in enumerate(lens):
        if n == 0:
            assert bool((out[b] == 0).all())
            continue
        c, s = cos[n - 1:n].double(), sin[n - 1:n].double()
        qr, _ = _turn(q[b].reshape(1, hq, d).double(), c, s)
        kr, ksize = _turn(k[b].reshape(1, hkv, d).double(), c, s)
        page, row = int(table[b, (n - 1) // ps]), (n - 1) % ps
        assert bool(((kp[page, :, row].double() - kr[0]).abs() <= half * kr[0].abs() + 3 * 2 ** -24 * ksize[0] + 1e-7).all())
        assert torch.equal(vp[page, :, row], v[b].reshape(hkv, d))
        pages = table[b, :-(-n // ps)].long()
        keys = kp[pages].transpose(0, 1).reshape(hkv, -1, d)[:, :n].double()
        values = vp[pages].transpose(0, 1).reshape(hkv, -1, d)[:, :n].double()
        qg = qr[0].view(hkv, hq // hkv, d)
        scores = qg @ keys.transpose(1, 2) / math.sqrt(d)
        size = (qg.abs() @ keys.abs().transpose(1, 2) / math.sqrt(d)).amax(-1, keepdim=True)
        p = torch.softmax(scores, -1)
        ref = p @ values
        move = 2 * size * (half + (d + 2) * 2 ** -24) + half + 2 ** -18 + n * 2 ** -24
        tol = move * (p @ values.abs()) + half * ref.abs() + 1e-7
        err = (out[b].view(hkv, hq // hkv, d).double() - ref).abs()
        assert bool((err <= tol).all()), (b, n, float((err / tol).max()))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens,hq,hkv,d,ps,fused", [
    ([1], 4, 1, 128, 16, False), ([2, 1, 0, 17], 8, 2, 128, 16, True), ([15, 16, 17, 31, 32, 33, 63, 64, 65, 66], 4, 2, 64, 16, False),
    ([129, 0, 300, 7], 32, 8, 128, 24, True), ([1000, 1, 5, 257], 5, 5, 64, 1, False), ([513, 64], 24, 1, 128, 64, True),
    ([3000], 64, 8, 128, 128, False), ([0, 0, 0], 4, 2, 128, 16, False), ([70, 71, 72, 73, 74, 75, 76] * 9, 16, 4, 64, 7, True),
    ([2049, 33], 20, 1, 64, 32, False), ([400], 33, 1, 128, 16, False), ([1, 200, 1, 1, 90, 1, 0, 1], 12, 4, 128, 100, False)])
def test_paged_attention(lens, hq, hkv, d, ps, fused, dtype):
    g = _gen(len(lens), hq, d, ps)
    kp, vp, table = _make_requests(lens, hkv, ps, d, dtype, g, interleaved=fused)
    q, k, v = _qkv_rows(len(lens), hq, hkv, d, dtype, g, fused)
    cos, sin = _tables_of_rotary(max(lens) + 1, d, dtype)
    pos = torch.tensor([n - 1 for n in lens], device=DEV)
    before = (kp.clone(), vp.clone())
    out = glue.paged_decode_attention(q, k, v, cos, sin, pos, table, kp, vp, hq, hkv, d)
    _check_attention(out, q, k, v, cos, sin, lens, table, kp, vp, hq, hkv, d, ps, dtype)
    # nothing but the new rows was written, and the same call gives the same bits
    for now, then in zip((kp, vp), before):
        now = now.clone()
        for b, n in enumerate(lens):
            if n:
                now[int(table[b, (n - 1) // ps]), :, (n - 1) % ps] = then[int(table[b, (n - 1) // ps]), :, (n - 1) % ps]
        assert torch.equal(now.view(torch.int16), then.view(torch.int16))
    assert torch.equal(out, glue.paged_decode_attention(q, k, v, cos, sin, pos, table, kp, vp, hq, hkv, d))


def test_paged_attention_of_large_scores_and_one_sided_weights():
    """Scores of several hundred: the running maximum moves a lot and most weights vanish; a single huge key takes all."""
    lens, hq, hkv, d, ps, dtype = [777, 130], 8, 2, 128, 16, torch.float16
    g = _gen(5, 5, 5)
    kp, vp, table = _make_requests(lens, hkv, ps, d, dtype, g)
    kp.mul_(8)
    q, k, v = _qkv_rows(2, hq, hkv, d, dtype, g, False)
    q, k = q * 8, k * 8
    cos, sin = _tables_of_rotary(800, d, dtype)
    out = glue.paged_decode_attention(q, k, v, cos, sin, torch.tensor([n - 1 for n in lens], device=DEV), table, kp, vp, hq, hkv, d)
    assert torch.isfinite(out).all()
    for b, n in enumerate(lens):                       # the exact weights at the rounded q (the tolerance above would be above 1 here)
        qr, _ = _turn(q[b].reshape(1, hq, d).double(), cos[n - 1:n].double(), sin[n - 1:n].double())
        pages = table[b, :-(-n // ps)].long()
        keys, values = (t[pages].transpose(0, 1).reshape(hkv, -1, d)[:, :n].double() for t in (kp, vp))
        qg = qr[0].to(dtype).double().view(hkv, hq // hkv, d)
        scores = qg @ keys.transpose(1, 2) / math.sqrt(d)
        size = (qg.abs() @ keys.abs().transpose(1, 2) / math.sqrt(d)).amax()
        p = torch.softmax(scores, -1)
        # q may have been rounded the other way where fp32 and fp64 rotation differ: one step of q in a few elements
        move = float(2 * size * (d + 2) * 2 ** -24) + 2 ** -10 + 2 ** -9 * 8 * 8 * 8 / math.sqrt(d)
        err = (out[b].view(hkv, hq // hkv, d).double() - p @ values).abs()
        assert bool((err <= move * (p @ values.abs()) + 2 ** -11 * (p @ values).abs() + 1e-6).all()), float(err.max())


def test_paged_attention_does_not_follow_bad_pages():
    lens, hq, hkv, d, ps, dtype = [40, 50, 20, 33, 10], 4, 2, 64, 8, torch.float16
    g = _gen(6, 6, 6)
    kp, vp, table = _make_requests(lens, hkv, ps, d, dtype, g)
    q, k, v = _qkv_rows(5, hq, hkv, d, dtype, g, False)
    cos, sin = _tables_of_rotary(60, d, dtype)
    pos = torch.tensor([n - 1 for n in lens], device=DEV)
    good = glue.paged_decode_attention(q, k, v, cos, sin, pos, table, kp, vp, hq, hkv, d)
    _lib.check_device_status()
    bad = table.clone()
    bad[0, 2], bad[1, 6], bad[3, 4] = kp.shape[0], -1, 1 << 30        # in the middle; of the new row; the last page
    pos2 = pos.clone()
    pos2[4] = 60                                                    # behind the cos / sin tables
    out = glue.paged_decode_attention(q, k, v, cos, sin, pos2, bad, kp, vp, hq, hkv, d)
    assert torch.isnan(out[[0, 1, 3, 4]]).all() and torch.equal(out[2], good[2])
    with pytest.raises(_lib.BitStackDeviceIndexError):
        _lib.check_device_status()
    pos2[4] = (table.shape[1]) * ps                                 # behind the table row
    long_cos, long_sin = _tables_of_rotary(4000, d, dtype)
    assert torch.isnan(glue.paged_decode_attention(q, k, v, long_cos, long_sin, pos2, table, kp, vp, hq, hkv, d)[4]).all()
    with pytest.raises(_lib.BitStackDeviceIndexError):
        _lib.check_device_status()


# ------------------------------------------------------------------------------------------------ sampling

def _ref_sample(x, u, t, k, p, mp):
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    if not np.max(x) > -np.inf:
        return 0, -np.inf
    if not t > 0:
        return int(np.argmax(x)), 0.0
    order = np.argsort(-x, kind="stable")
    top = x[order[0]]
    with np.errstate(invalid="ignore", over="ignore"):
        z = (x - top) * (1.0 / np.float64(t))
    w = np.exp(np.where(x == top, 0.0, np.where(np.isnan(z), -np.inf, z)))
    # The sums in integers of 2^-44: a running float64 sum rounds, and calls a border that u (or p) meets exactly the wrong
    # way (0, 1, 2, 0, 1, 2, ... at u = 1/2: sums[299] came out above half the total that it equals).  Quantising moves a
    # border by at most V 2^-45 of the largest weight, which only a u that near to a border would notice.
    w = np.rint(np.ldexp(w, 44)).astype(np.int64)
    n = len(x) if k <= 0 else min(k, len(x))
    if p < 1:
        sums = np.cumsum(w[order[:n]])
        want = math.ceil(Fraction(float(p)) * int(sums[-1]))          # sums < want, exactly
        n = min(n, 1 + int(np.searchsorted(sums, want, side="left")))
    if mp > 0:
        n = max(1, int(np.sum(w[order[:n]] >= min(mp, 1.0) * 2.0 ** 44)))
    kept = np.sort(order[:n])
    sums = np.cumsum(w[kept])
    want = math.floor(Fraction(float(u if u > 0 else 0.0)) * int(sums[-1]))   # sums > want, exactly
    at = min(int(np.searchsorted(sums, want, side="right")), n - 1)
    return int(kept[at]), float(z[kept[at]] if x[kept[at]] != top else 0.0) - math.log(int(sums[-1]) / 2 ** 44)


def _check_sample(logits, u, **kw):
    B = logits.shape[0]
    tokens = torch.full((B,), -1, dtype=torch.int64, device=DEV)
    lp = torch.full((B,), 7.0, device=DEV)
    dev = {n: None if a is None else torch.tensor(a, dtype=torch.int32 if n == "top_k" else torch.float32, device=DEV) for n, a in kw.items()}
    got = glue.sample_step(logits, u, tokens, logprobs=lp, **dev)
    assert got is tokens
    x, uu = logits.float().cpu().numpy(), u.double().cpu().numpy()
    for b in range(B):
        set_ = lambda n, off, t: off if kw.get(n) is None else t(dev[n][b].item())  # noqa: E731
        want, want_lp = _ref_sample(x[b], uu[b], set_("temperature", 1.0, float), set_("top_k", 0, int), set_("top_p", 1.0, float), set_("min_p", 0.0, float))
        assert int(tokens[b]) == want, (b, int(tokens[b]), want)
        if math.isinf(want_lp):
            assert float(lp[b]) == want_lp
        else:                                          # one rounding to fp32, and the fixed-point weights' 2^-40
            assert abs(float(lp[b]) - want_lp) <= 2 ** -23 * abs(want_lp) + 1e-7
    return tokens


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,V", [(1, 1), (3, 2), (4, 7), (5, 257), (6, 1000), (3, 4099), (7, 32000), (2, 50257), (2, 128256), (1, 262144)])
def test_sample_step(B, V, dtype):
    g = _gen(B, V)
    x = torch.randn(B, V + 3, device=DEV, generator=g) * 3
    x[:, :V].scatter_add_(1, torch.randint(0, V, (B, 5), device=DEV, generator=g), torch.full((B, 5), 6.0, device=DEV))
    logits = x.to(dtype)[:, :V]                        # rows that are not 16-byte aligned
    u = torch.rand(B, device=DEV, generator=g)
    _check_sample(logits, u)
    _check_sample(logits, u, temperature=[0.7] * B, top_k=[min(V, 40)] * B)
    _check_sample(logits, u, temperature=[1.3] * B, top_p=[0.9] * B)
    _check_sample(logits, u, min_p=[0.05] * B)
    _check_sample(logits.contiguous(), u, temperature=[(0.0, 0.5, 1.0, 2.0)[b % 4] for b in range(B)], top_k=[(0, 1, V // 2, 5, V + 9)[b % 5] for b in range(B)],
                  top_p=[(0.3, 1.0, 0.95)[b % 3] for b in range(B)], min_p=[(0.0, 0.2)[b % 2] for b in range(B)])


@pytest.mark.parametrize("u", [0.0, 2.0 ** -24, 0.5, 0.999, 1 - 2.0 ** -24])
def test_sample_step_ties_and_borders(u):
    """Many equal logits (ties go to the lowest index), borders that the uniform number hits exactly."""
    V = 600
    rows = torch.zeros(6, V, device=DEV)
    rows[1] = torch.arange(V, device=DEV) % 3
    rows[2, 100:] = -math.inf
    rows[3, ::2] = -0.0
    rows[4] = -1e30
    rows[4, 17] = 5
    rows[5] = torch.arange(V, 0, -1, device=DEV) * 0.001
    uu = torch.full((6,), u, device=DEV)
    for kw in (dict(), dict(top_k=[7] * 6), dict(top_p=[0.5] * 6), dict(top_p=[0.25] * 6, top_k=[64] * 6), dict(min_p=[1.0] * 6), dict(min_p=[7.0] * 6),
               dict(top_p=[0.0] * 6), dict(top_p=[-1.0] * 6), dict(top_k=[V] * 6), dict(top_k=[-3] * 6), dict(top_p=[1.0] * 6), dict(top_p=[1 - 2.0 ** -24] * 6)):
        _check_sample(rows.half(), uu, **kw)
        _check_sample(rows, uu, **kw)


def test_sample_step_of_odd_values():
    V = 300
    x = torch.randn(10, V, device=DEV, generator=_gen(8)) * 2
    x[0] = -math.inf                                   # a mask that leaves nothing
    x[1] = math.nan
    x[2, 5:] = math.nan
    x[3, [9, 200]] = math.inf                          # infinities share everything
    x[4, ::3] = -math.inf
    u = torch.tensor([.3, .3, .9, .7, .5, math.nan, 1.0, 2.0, -1.0, .99], device=DEV)
    ref_u = torch.tensor([.3, .3, .9, .7, .5, 0.0, 1 - 2.0 ** -24, 1 - 2.0 ** -24, 0.0, .99], device=DEV)
    for kw in (dict(), dict(temperature=[1e-30] * 10), dict(temperature=[math.inf] * 10), dict(temperature=[math.nan] * 10), dict(temperature=[-1.0] * 10),
               dict(temperature=[1e-42] * 10), dict(top_p=[math.nan] * 10), dict(min_p=[math.nan] * 10), dict(top_p=[0.9] * 10, top_k=[250] * 10)):
        a = _check_sample(x, ref_u, **kw)
        tokens = torch.zeros(10, dtype=torch.int64, device=DEV)
        dev = {n: torch.tensor(v, dtype=torch.int32 if n == "top_k" else torch.float32, device=DEV) for n, v in kw.items()}
        assert torch.equal(a, glue.sample_step(x, u, tokens, **dev))


def test_sample_step_moves_the_position_and_greedy_rows_are_the_greedy_step():
    x = (torch.randn(4, 32001, device=DEV, generator=_gen(9)) * 2).half()
    a, b = torch.zeros(4, dtype=torch.int64, device=DEV), torch.zeros(4, dtype=torch.int64, device=DEV)
    pos = torch.tensor([7], device=DEV)
    glue.sample_step(x, torch.rand(4, device=DEV), a, torch.zeros(4, device=DEV), pos=pos)
    assert torch.equal(a, glue.greedy_step(x, b, None)) and pos.item() == 8


def test_sample_step_frequencies():
    """8192 evenly spread numbers: every kept token comes as often as its probability says, to within one."""
    n, V = 8192, 50
    x = torch.randn(1, V, device=DEV, generator=_gen(10)) * 2
    u = (torch.arange(n, device=DEV) + 0.5) / n
    tokens = torch.zeros(n, dtype=torch.int64, device=DEV)
    glue.sample_step(x.repeat(n, 1), u, tokens)
    assert bool(((tokens.bincount(minlength=V) - torch.softmax(x[0].double(), 0) * n).abs() <= 1.0001).all())


# ------------------------------------------------------------------------------------------------ calls side by side

def test_more_requests_than_one_launch_takes():
    """4100 requests: three launches on one scratch, idle rows and one-token requests among them."""
    g = _gen(4, 1, 0, 0)
    lens = torch.randint(0, 40, (4100,), generator=torch.Generator().manual_seed(4)).tolist()
    hq, hkv, d, ps, dtype = 2, 1, 64, 16, torch.float16
    kp, vp, table = _make_requests(lens, hkv, ps, d, dtype, g, poison=False)
    table = torch.cat([table, torch.full((4100, 40), -1, dtype=torch.int32, device=DEV)], 1)   # wide enough for the shared form
    q, k, v = _qkv_rows(4100, hq, hkv, d, dtype, g, False)
    cos, sin = _tables_of_rotary(41, d, dtype)
    out = glue.paged_decode_attention(q, k, v, cos, sin, torch.tensor([n - 1 for n in lens], device=DEV), table, kp, vp, hq, hkv, d)
    some = list(range(0, 4100, 97)) + [2047, 2048, 4095, 4096, 4099]
    at = torch.tensor(some, device=DEV)
    _check_attention(out[at], q[at], k[at], v[at], cos, sin, [lens[i] for i in some], table[at], kp, vp, hq, hkv, d, ps, dtype)


def test_calls_on_several_streams_at_once():
    """Attention and sampling on four streams at the same time, each with scratch of its own: the results of one after the other."""
    jobs = []
    for i in range(4):
        g = _gen(9, i)
        lens, hq, hkv, d, ps, dtype = [900 + 100 * i, 40, 0, 613], 8, 2, 128, 16, torch.float16
        kp, vp, table = _make_requests(lens, hkv, ps, d, dtype, g)
        q, k, v = _qkv_rows(4, hq, hkv, d, dtype, g, False)
        cos, sin = _tables_of_rotary(1300, d, dtype)
        pos = torch.tensor([n - 1 for n in lens], device=DEV)
        logits = torch.randn(5, 30000, device=DEV, generator=g)
        u, p = torch.rand(5, device=DEV, generator=g), torch.full((5,), 0.9, device=DEV)
        jobs.append((q, k, v, cos, sin, pos, table, kp, vp, hq, hkv, d, logits, u, p))

    def run(j):
        return (glue.paged_decode_attention(*j[:12]), glue.sample_step(j[12], j[13], torch.zeros(5, dtype=torch.int64, device=DEV), top_p=j[14]))
    want = [run(j) for j in jobs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in jobs], [[] for _ in jobs]
    for _ in range(20):
        for i, (j, s) in enumerate(zip(jobs, streams)):
            with torch.cuda.stream(s):
                got[i].append(run(j))
    torch.cuda.synchronize()
    for w, gs in zip(want, got):
        assert all(torch.equal(a, b) for r in gs for a, b in zip(r, w))


def test_table_rows_that_several_requests_share():
    """A common prefix: pages that two requests' rows both list are read by both (each writes a page of its own)."""
    g, hq, hkv, d, ps, dtype = _gen(3, 3), 4, 2, 64, 8, torch.float16
    kp, vp = _pool(12, hkv, ps, d, dtype, g, False)
    table = torch.tensor([[3, 5, 7, 1], [3, 5, 7, 2], [3, 5, 7, 9]], dtype=torch.int32, device=DEV)
    q, k, v = _qkv_rows(3, hq, hkv, d, dtype, g, False)
    cos, sin = _tables_of_rotary(32, d, dtype)
    lens = [25, 30, 32]
    out = glue.paged_decode_attention(q, k, v, cos, sin, torch.tensor([n - 1 for n in lens], device=DEV), table, kp, vp, hq, hkv, d)
    _check_attention(out, q, k, v, cos, sin, lens, table, kp, vp, hq, hkv, d, ps, dtype)


def test_wrong_arguments_on_the_device():
    x = torch.zeros(2, 128, device=DEV, dtype=torch.float16)
    pool, i = torch.zeros(4, 1, 8, 128, device=DEV, dtype=torch.float16), torch.zeros(2, 3, dtype=torch.int32, device=DEV)
    pos = torch.full((2,), -1, device=DEV)
    ok = dict(q=x, k=x, v=x, cos=x, sin=x, positions=pos, block_table=i, k_pages=pool, v_pages=pool, q_heads=1, kv_heads=1, head_dim=128)
    assert bool((glue.paged_decode_attention(**ok) == 0).all())
    for bad in (dict(k=x[:1]), dict(v=x.bfloat16()), dict(positions=pos.int()), dict(block_table=i.long()), dict(block_table=i[:1]), dict(cos=x[:, :64]),
                dict(k_pages=pool[:, :, :, :64]), dict(v_pages=pool[:3]), dict(k_pages=pool.transpose(0, 2)), dict(q=x.t()), dict(q_heads=2),
                dict(k_pages=pool.expand(4, 1, 8, 128)[:, :, :0]), dict(k_pages=pool[:1].expand(4, 1, 8, 128)), dict(positions=pos.cpu()), dict(kv_heads=0)):
        with pytest.raises(ValueError):
            glue.paged_decode_attention(**{**ok, **bad})
    lo, u, t = torch.zeros(2, 9, device=DEV), torch.zeros(2, device=DEV), torch.zeros(2, dtype=torch.int64, device=DEV)
    for bad in (dict(uniforms=u[:1]), dict(tokens=t.int()), dict(temperature=u.double()), dict(top_k=u), dict(top_p=u[:1]), dict(pos=t), dict(logits=lo.t()),
                dict(logits=lo[:1].expand(2, 9)), dict(logprobs=u.cpu())):
        with pytest.raises(ValueError):
            glue.sample_step(**{**dict(logits=lo, uniforms=u, tokens=t), **bad})
    n, c = torch.zeros(2, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    for bad in (dict(page_size=0), dict(page_size=1 << 40), dict(max_tokens=-1), dict(free_count=n), dict(lens_out=c), dict(new_tokens=n.long()), dict(free_pages=c[:0])):
        with pytest.raises(ValueError):
            glue.page_tables(**{**dict(lens=n, new_tokens=n, block_table=i, free_pages=c, free_count=c, page_size=4), **bad})


def test_pages_as_a_dense_cache():
    """One page per request is the dense cache's layout: a prompt written by the paged call, then read by the dense decode
    attention directly behind it, and the other way round."""
    g, B, hq, hkv, d, L = _gen(11, 2), 3, 8, 2, 128, 700
    cos, sin = _tables_of_rotary(L, d, torch.float16)
    for _ in range(20):
        kc, vc = (torch.zeros(B, hkv, L, d, device=DEV, dtype=torch.float16) for _ in range(2))
        n = 650
        q, k, v = _qkv_rows(B * n, hq, hkv, d, torch.float16, g, False)
        pos = torch.arange(n, device=DEV).repeat(B)
        slots = pos + torch.arange(B, device=DEV).repeat_interleave(n) * L
        q1, k1, v1 = _qkv_rows(B, hq, hkv, d, torch.float16, g, False)
        at = torch.tensor([n], device=DEV)
        torch.cuda.synchronize()
        glue.rope_paged_cache(q, k, v, cos, sin, pos, slots, kc, vc, hq, hkv, d)
        dense = glue.decode_attention(q1, k1, v1, cos, sin, at, kc, vc, hq, hkv, d)
        table = torch.arange(B, device=DEV, dtype=torch.int32).view(B, 1)
        paged = glue.paged_decode_attention(q1, k1, v1, cos, sin, at.repeat(B), table, kc, vc, hq, hkv, d)
        _check_attention(paged, q1, k1, v1, cos, sin, [n + 1] * B, table, kc, vc, hq, hkv, d, L, torch.float16)
        # the dense call rounds q after its rotation too, accumulates in fp32 and sums 2^-18 off at most: the same bound
        _check_attention(dense, q1, k1, v1, cos, sin, [n + 1] * B, table, kc, vc, hq, hkv, d, L, torch.float16)
