"""What the serving operators refuse, on the host and without a GPU: arguments are checked before anything is launched."""
import ctypes as C

import pytest
import torch

from bitstack_b200 import _lib, glue

ANY = 1 << 20   # a non-null, aligned address: refused calls never follow it


@pytest.fixture(scope="module")
def lib():
    from bitstack_b200.build import build, build_serving
    build()
    build_serving()
    return _lib.load()


def _tables(lib, **kw):
    a = dict(batch=4, stride=8, width=8, capacity=16, page=16, tokens=4, slots=ANY, offsets=ANY)
    a.update(kw)
    return lib.bsb_page_tables(ANY, ANY, a["batch"], ANY, a["stride"], a["width"], ANY, ANY, a["capacity"], a["page"], a["tokens"], a["slots"], ANY,
                               a["offsets"], ANY, ANY, ANY, None)


@pytest.mark.parametrize("kw,code", [(dict(batch=0), -1), (dict(stride=7), -1), (dict(width=0), -1), (dict(page=0), -1), (dict(capacity=0), -1),
                                     (dict(tokens=-1), -1), (dict(slots=None), -1), (dict(offsets=None), -1), (dict(batch=8193), -4)])
def test_page_tables(lib, kw, code):
    assert _tables(lib, **kw) == code and lib.bsb_last_error()


@pytest.mark.parametrize("kw,code", [(dict(batch=0), -1), (dict(batch=8193), -4), (dict(done=None), -1), (dict(page=0), -1)])
def test_release_pages(lib, kw, code):
    a = dict(batch=4, done=ANY, page=16)
    a.update(kw)
    assert lib.bsb_release_pages(a["done"], ANY, a["batch"], ANY, 8, 8, ANY, ANY, 16, a["page"], None) == code


def _write(lib, **kw):
    a = dict(q=ANY, qs=512, ks=256, vs=256, tl=64, np=8, kps=2 * 16 * 128, vps=2 * 16 * 128, tokens=3, hq=4, hkv=2, d=128, page=16, dtype=0)
    a.update(kw)
    return lib.bsb_rope_paged_cache(a["q"], ANY, ANY, a["qs"], a["ks"], a["vs"], ANY, ANY, a["tl"], ANY, ANY, ANY, ANY, ANY, a["np"], a["kps"],
                                    a["vps"], a["tokens"], a["hq"], a["hkv"], a["d"], a["page"], a["dtype"], None)


def _attend(lib, **kw):
    a = dict(q=ANY, qs=512, ks=256, vs=256, tl=64, ts=4, tw=4, np=8, kps=2 * 16 * 128, vps=2 * 16 * 128, batch=3, hq=4, hkv=2, d=128, page=16, dtype=0,
             sc=ANY, scb=1 << 40)
    a.update(kw)
    return lib.bsb_paged_decode_attention(a["q"], ANY, ANY, a["qs"], a["ks"], a["vs"], ANY, ANY, a["tl"], ANY, ANY, a["ts"], a["tw"], ANY, ANY, a["np"],
                                          a["kps"], a["vps"], ANY, a["batch"], a["hq"], a["hkv"], a["d"], a["page"], a["dtype"], a["sc"], a["scb"], None)


_BOTH = [dict(q=None), dict(q=ANY + 8), dict(qs=504), dict(qs=516), dict(ks=248), dict(vs=252), dict(tl=0), dict(np=0), dict(kps=2 * 16 * 128 - 8),
         dict(vps=2 * 16 * 128 + 4), dict(hq=0), dict(hkv=0), dict(page=0), dict(dtype=2), dict(dtype=9)]


@pytest.mark.parametrize("kw", _BOTH + [dict(d=24), dict(d=0), dict(d=528), dict(tokens=-1)])
def test_rope_paged_cache(lib, kw):
    assert _write(lib, **kw) == -1 and lib.bsb_last_error()


@pytest.mark.parametrize("kw", _BOTH + [dict(d=96), dict(d=256), dict(hq=5), dict(ts=3), dict(tw=0), dict(batch=-1), dict(np=1 << 31)])
def test_paged_attention(lib, kw):
    assert _attend(lib, **kw) == -1 and lib.bsb_last_error()
    assert _attend(lib, batch=1 << 30) == -1
    assert _attend(lib, scb=16) == -3 and _attend(lib, sc=None) == -1 and _attend(lib, sc=ANY + 8) == -1


@pytest.mark.parametrize("kw,code", [(dict(vocab=0), -1), (dict(stride=9), -1), (dict(dtype=3), -1), (dict(logits=None), -1), (dict(u=None), -1),
                                     (dict(tokens=None), -1), (dict(batch=-1), -1), (dict(batch=(1 << 24) + 1), -4), (dict(vocab=262145, stride=1 << 21), -4)])
def test_sample_step(lib, kw, code):
    a = dict(logits=ANY, batch=2, vocab=10, stride=10, dtype=0, u=ANY, tokens=ANY)
    a.update(kw)
    assert lib.bsb_sample_step(a["logits"], a["batch"], a["vocab"], a["stride"], a["dtype"], a["u"], None, None, None, None, a["tokens"], None, None,
                               None) == code


def test_nothing_to_do_is_fine(lib):
    assert _write(lib, tokens=0) == 0 and _attend(lib, batch=0) == 0
    assert lib.bsb_sample_step(ANY, 0, 10, 10, 0, ANY, None, None, None, None, ANY, None, None, None) == 0
    assert lib.bsb_paged_attention_scratch_bytes(4, 32, 8, 128) >= 0
    assert lib.bsb_paged_attention_scratch_bytes(4, 5, 2, 128) == -1


def test_wrappers_refuse_host_tensors(lib):
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        glue.page_tables(i, i, torch.zeros(2, 3, dtype=torch.int32), i, torch.zeros(1, dtype=torch.int32), 16)
    with pytest.raises(ValueError, match="CUDA"):
        glue.release_pages(torch.zeros(2, dtype=torch.bool), i, torch.zeros(2, 3, dtype=torch.int32), i, i[:1], 16)
    with pytest.raises(ValueError, match="CUDA"):
        glue.sample_step(torch.zeros(2, 5).half(), torch.zeros(2), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="fp16, bf16 or fp32"):
        glue.sample_step(torch.zeros(2, 5).double(), torch.zeros(2), torch.zeros(2, dtype=torch.int64))
    x = torch.zeros(2, 128).half()
    for call in (glue.rope_paged_cache, glue.paged_decode_attention):
        with pytest.raises(ValueError, match="CUDA"):
            call(x, x, x, x, x, i.long(), i.long(), x, x, 1, 1, 128)
        with pytest.raises(ValueError, match="fp16 or bf16"):
            call(x.float(), x, x, x, x, i.long(), i.long(), x, x, 1, 1, 128)


def test_bad_indices_have_an_error_of_their_own(monkeypatch):
    class Fake:
        def bsb_read_status(self, code, clear):
            return -6

        def bsb_last_error(self):
            return b"a kernel met an index outside its tensor"
    monkeypatch.setattr(_lib, "_lib", Fake())
    with pytest.raises(_lib.BitStackDeviceIndexError, match="outside"):
        _lib.check_device_status()
    assert issubclass(_lib.BitStackDeviceIndexError, _lib.BitStackLibraryError) and C.sizeof(C.c_int32) == 4
