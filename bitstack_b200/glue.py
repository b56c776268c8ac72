"""Fused decode-time glue ops (residual add + RMSNorm, rotary + KV-cache write, SiLU*up) on CUDA
tensors, through the C ABI.  These are harness helpers around the BitStack projections; the
reference leaves the same ops to the Hugging Face Llama modules."""
from __future__ import annotations

import torch

from . import _lib


_att_scratch = {}   # (device, batch, heads, head_dim) -> zero-initialised scratch of decode_attention


def _s(t):
    return torch.cuda.current_stream(t.device).cuda_stream


def add_rmsnorm(h: torch.Tensor, delta, weight: torch.Tensor, eps: float, absmax: torch.Tensor = None) -> torch.Tensor:
    """In place h += delta (skipped when delta is None); returns rmsnorm(h) * weight.  h: [rows, hidden] fp16.
    `absmax` (fp32 [rows], optional) receives max |result| per row."""
    assert h.is_cuda and h.dtype == torch.float16 and h.is_contiguous() and h.dim() == 2
    if delta is not None:
        delta = delta.reshape(h.shape)
        assert delta.dtype == torch.float16 and delta.is_contiguous()
    if absmax is not None:
        assert absmax.dtype == torch.float32 and absmax.is_contiguous() and absmax.numel() >= h.shape[0]
    y = torch.empty_like(h)
    with torch.cuda.device(h.device):
        rc = _lib.load().bsb_add_rmsnorm(h.data_ptr(), None if delta is None else delta.data_ptr(), weight.data_ptr(),
                                         float(eps), y.data_ptr(), None if absmax is None else absmax.data_ptr(),
                                         h.shape[0], h.shape[1], _s(h))
    _lib.check(rc, "bsb_add_rmsnorm")
    return y


def rope_cache(q, k, v, cos, sin, pos, k_cache, v_cache, q_heads, kv_heads, head_dim):
    """Rotary embedding at position pos[0] (device int64) on q in place and on k, which goes with v
    into k_cache / v_cache [batch, kv_heads, max_len, head_dim]."""
    for t in (q, k, v, cos, sin, k_cache, v_cache):
        assert t.is_cuda and t.dtype == torch.float16 and t.is_contiguous()
    assert pos.dtype == torch.int64 and pos.is_cuda
    batch = q.shape[0]
    with torch.cuda.device(q.device):
        rc = _lib.load().bsb_rope_cache(q.data_ptr(), k.data_ptr(), v.data_ptr(), cos.data_ptr(), sin.data_ptr(),
                                        pos.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), batch, q_heads, kv_heads,
                                        head_dim, k_cache.shape[2], _s(q))
    _lib.check(rc, "bsb_rope_cache")
    return q


def decode_attention(q, k, v, cos, sin, pos, k_cache, v_cache, q_heads, kv_heads, head_dim):
    """One new token per batch row: rotary embedding of q and k at position pos[0] (device int64), k and v
    appended to k_cache / v_cache [batch, kv_heads, max_len, head_dim], then grouped-query attention of the
    rotated q over cache positions 0..pos.  q is left untouched; returns [batch, q_heads * head_dim] fp16."""
    for t in (q, k, v, cos, sin, k_cache, v_cache):
        assert t.is_cuda and t.dtype == torch.float16 and t.is_contiguous()
    assert pos.dtype == torch.int64 and pos.is_cuda
    batch = q.shape[0]
    out = torch.empty(batch, q_heads * head_dim, dtype=torch.float16, device=q.device)
    lib = _lib.load()
    key = (q.device.index, batch, q_heads, head_dim)
    scratch = _att_scratch.get(key)
    if scratch is None:   # zeroed once; the kernel leaves its counters at zero for the next call
        scratch = torch.zeros(lib.bsb_decode_attention_scratch_bytes(batch, q_heads, head_dim), dtype=torch.uint8, device=q.device)
        _att_scratch[key] = scratch
    with torch.cuda.device(q.device):
        rc = lib.bsb_decode_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), cos.data_ptr(), sin.data_ptr(),
                                      pos.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), batch,
                                      q_heads, kv_heads, head_dim, k_cache.shape[2], scratch.data_ptr(), scratch.numel(), _s(q))
    _lib.check(rc, "bsb_decode_attention")
    return out


def greedy_step(logits: torch.Tensor, tokens: torch.Tensor, pos) -> torch.Tensor:
    """tokens[b] = argmax(logits[b]) (first maximum), then pos[0] += 1 (skipped when pos is None), in one launch.
    logits: [batch, vocab] fp16 with unit inner stride; tokens: [batch] int64; pos: [1] int64 or None."""
    assert logits.is_cuda and logits.dtype == torch.float16 and logits.dim() == 2 and logits.stride(1) == 1
    assert tokens.dtype == torch.int64 and tokens.is_contiguous() and tokens.numel() == logits.shape[0]
    assert pos is None or (pos.dtype == torch.int64 and pos.is_cuda)
    with torch.cuda.device(logits.device):
        rc = _lib.load().bsb_greedy_step(logits.data_ptr(), logits.shape[0], logits.shape[1], logits.stride(0), tokens.data_ptr(),
                                         None if pos is None else pos.data_ptr(), _s(logits))
    _lib.check(rc, "bsb_greedy_step")
    return tokens


def silu_mul(gate: torch.Tensor, up: torch.Tensor, absmax: torch.Tensor = None) -> torch.Tensor:
    """silu(gate) * up on [rows, n] fp16 (n % 8 == 0); `absmax` (fp32 [rows], optional) receives max |result| per row."""
    assert gate.is_cuda and gate.dtype == torch.float16 and gate.is_contiguous() and up.is_contiguous()
    g2 = gate.reshape(-1, gate.shape[-1])
    out = torch.empty_like(gate)
    with torch.cuda.device(gate.device):
        rc = _lib.load().bsb_silu_mul(gate.data_ptr(), up.data_ptr(), out.data_ptr(),
                                      None if absmax is None else absmax.data_ptr(), g2.shape[0], g2.shape[1], _s(gate))
    _lib.check(rc, "bsb_silu_mul")
    return out


# ---------------------------------------------------------------------------------- serving over a paged cache
# These calls are a few microseconds of GPU work at small sizes, so the wrappers are written for the host's time: one
# comparison per tensor where it is as it should be, and the explanations only where it is not.
_DTYPES = {torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16, torch.float32: _lib.DTYPE_F32}
_raw_stream = torch._C._cuda_getCurrentRawStream


def _need(t, name: str, dtype, shape, index: int, strided: bool = False) -> None:
    """Raises ValueError unless `t` is a CUDA tensor on device `index` of this type and shape (None = any extent),
    contiguous, or with `strided` only in its last dimension."""
    if type(t) is torch.Tensor and t.dtype is dtype and t.get_device() == index and t.shape == shape and t.is_contiguous():
        return
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.get_device() != index:
        raise ValueError(f"{name} must be a CUDA tensor on cuda:{max(index, 0)}")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if t.dim() != len(shape) or any(w is not None and n != w for n, w in zip(t.shape, shape)):
        raise ValueError(f"{name} must have shape {['any' if w is None else w for w in shape]}, got {list(t.shape)}")
    if not (t.is_contiguous() or (strided and (t.shape[-1] <= 1 or t.stride(-1) == 1))):
        raise ValueError(f"{name} must be contiguous" + (" in its last dimension" if strided else ""))


def _index(t, name: str) -> int:
    """Device index of a call's first tensor."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    return t.get_device()


def _launch(what: str, index: int, *args) -> None:
    """Calls the library's `what` on the current stream of device `index`, with that device current."""
    fn = getattr(_lib.load(), what)
    if torch.cuda.current_device() == index:
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc != 0:
        _lib.check(rc, what)


def _row_stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _pages(k_pages, v_pages, dtype, kv_heads, head_dim, index):
    """(num_pages, page_size, strides of a page) of a cache [num_pages, kv_heads, page_size, head_dim] whose pages are
    contiguous; the pages themselves may lie apart (one allocation that interleaves K and V, or the layers)."""
    _need(k_pages, "k_pages", dtype, (None, kv_heads, None, head_dim), index, True)
    shape = k_pages.shape
    _need(v_pages, "v_pages", dtype, shape, index, True)
    n, _, ps, _ = shape
    if n < 1 or ps < 1:
        raise ValueError("the page pool is empty")
    inner = kv_heads * ps * head_dim
    if k_pages.is_contiguous() and v_pages.is_contiguous():
        return n, ps, inner, inner
    for t, name in ((k_pages, "k_pages"), (v_pages, "v_pages")):
        if not t[0].is_contiguous() or (n > 1 and t.stride(0) < inner):
            raise ValueError(f"{name}: every page [kv_heads, page_size, head_dim] must be contiguous and apart from the next")
    return n, ps, k_pages.stride(0) if n > 1 else inner, v_pages.stride(0) if n > 1 else inner


def _page_lists(lens, block_table, free_pages, free_count):
    """(device index, requests, width of the table) of the bookkeeping tensors."""
    index = _index(lens, "lens")
    batch = lens.shape[0] if lens.dim() == 1 else 0
    _need(lens, "lens", torch.int32, (batch,), index)
    width = block_table.shape[-1] if isinstance(block_table, torch.Tensor) and block_table.dim() else 0
    _need(block_table, "block_table", torch.int32, (batch, width), index, True)
    _need(free_pages, "free_pages", torch.int32, (None,), index)
    _need(free_count, "free_count", torch.int32, (1,), index)
    return index, batch, width


def page_tables(lens, new_tokens, block_table, free_pages, free_count, page_size: int, max_tokens: int = 0, lens_out=None, free_count_out=None):
    """One step of a paged cache's bookkeeping on the device: request b holds lens[b] tokens (int32 [batch]) and gets
    new_tokens[b] more; pages it lacks are popped from the stack free_pages[:free_count] and entered in its row of
    block_table (int32 [batch, width], updated in place).  lens and free_count (int32 [1]) are updated in place unless
    lens_out / free_count_out receive the new values.  A request whose row is too narrow, or for which the stack runs out
    (requests in order), is refused: it keeps its length.

    Returns (slots, positions, offsets, last): slot and position of every new token, request after request, int64
    [max_tokens], -1 for tokens of refused requests and behind the end; int32 [batch + 1] first token of every request;
    int64 [batch] position of the request's last new token, -1 when it has none or was refused."""
    index, batch, width = _page_lists(lens, block_table, free_pages, free_count)
    _need(new_tokens, "new_tokens", torch.int32, (batch,), index)
    if lens_out is None:
        lens_out = lens
    else:
        _need(lens_out, "lens_out", torch.int32, (batch,), index)
    if free_count_out is None:
        free_count_out = free_count
    else:
        _need(free_count_out, "free_count_out", torch.int32, (1,), index)
    if max_tokens < 0:
        raise ValueError("max_tokens must not be negative")
    dev = lens.device
    slots = torch.empty(max_tokens, dtype=torch.int64, device=dev)
    positions = torch.empty(max_tokens, dtype=torch.int64, device=dev)
    offsets = torch.empty(batch + 1, dtype=torch.int32, device=dev)
    last = torch.empty(batch, dtype=torch.int64, device=dev)
    _launch("bsb_page_tables", index, lens.data_ptr(), new_tokens.data_ptr(), batch, block_table.data_ptr(), _row_stride(block_table), width,
            free_pages.data_ptr(), free_count.data_ptr(), free_pages.shape[0], page_size, max_tokens, slots.data_ptr(), positions.data_ptr(),
            offsets.data_ptr(), last.data_ptr(), lens_out.data_ptr(), free_count_out.data_ptr())
    return slots, positions, offsets, last


def release_pages(done, lens, block_table, free_pages, free_count, page_size: int) -> None:
    """Requests with done[b] (bool [batch]) give their pages back to the stack, and their length becomes 0 (in place)."""
    index, batch, width = _page_lists(lens, block_table, free_pages, free_count)
    _need(done, "done", torch.bool, (batch,), index)
    _launch("bsb_release_pages", index, done.data_ptr(), lens.data_ptr(), batch, block_table.data_ptr(), _row_stride(block_table), width,
            free_pages.data_ptr(), free_count.data_ptr(), free_pages.shape[0], page_size)


def _qkv(q, k, v, cos, sin, q_heads, kv_heads, head_dim):
    dtype = q.dtype if isinstance(q, torch.Tensor) else None
    if dtype is not torch.float16 and dtype is not torch.bfloat16:
        raise ValueError(f"q must be fp16 or bf16, got {dtype}")
    index = _index(q, "q")
    rows = q.shape[0] if q.dim() else 0
    _need(q, "q", dtype, (rows, q_heads * head_dim), index, True)
    _need(k, "k", dtype, (rows, kv_heads * head_dim), index, True)
    _need(v, "v", dtype, (rows, kv_heads * head_dim), index, True)
    _need(cos, "cos", dtype, (None, head_dim) if not isinstance(cos, torch.Tensor) or cos.dim() != 2 else (cos.shape[0], head_dim), index)
    _need(sin, "sin", dtype, cos.shape, index)
    return index, dtype, rows


def rope_paged_cache(q, k, v, cos, sin, positions, slots, k_pages, v_pages, q_heads, kv_heads, head_dim):
    """Rotary embedding of a batch of tokens (a prompt, or several requests' tokens) at `positions` (int64 [tokens]); k and v
    go to `slots` (int64 [tokens]) of k_pages / v_pages [num_pages, kv_heads, page_size, head_dim].  Returns the rotated q
    [tokens, q_heads * head_dim].  Position -1: padding (its q row is 0, nothing is cached); slot -1: not cached."""
    index, dtype, rows = _qkv(q, k, v, cos, sin, q_heads, kv_heads, head_dim)
    n, ps, ks, vs = _pages(k_pages, v_pages, dtype, kv_heads, head_dim, index)
    _need(positions, "positions", torch.int64, (rows,), index)
    _need(slots, "slots", torch.int64, (rows,), index)
    out = torch.empty(rows, q_heads * head_dim, dtype=dtype, device=q.device)
    _launch("bsb_rope_paged_cache", index, q.data_ptr(), k.data_ptr(), v.data_ptr(), _row_stride(q), _row_stride(k), _row_stride(v),
            cos.data_ptr(), sin.data_ptr(), cos.shape[0], positions.data_ptr(), slots.data_ptr(), out.data_ptr(), k_pages.data_ptr(),
            v_pages.data_ptr(), n, ks, vs, rows, q_heads, kv_heads, head_dim, ps, _DTYPES[dtype])
    return out


def paged_decode_attention(q, k, v, cos, sin, positions, block_table, k_pages, v_pages, q_heads, kv_heads, head_dim):
    """One new token per request at positions[b] (int64 [batch]; -1: idle row): rotary embedding of q and k, k and v written
    into the request's page (block_table int32 [batch, width]), then grouped-query attention over positions 0 .. positions[b].
    q, k, v: [batch, heads * head_dim], rows may be strided views; fp16 or bf16.  Returns [batch, q_heads * head_dim]."""
    index, dtype, rows = _qkv(q, k, v, cos, sin, q_heads, kv_heads, head_dim)
    n, ps, ks, vs = _pages(k_pages, v_pages, dtype, kv_heads, head_dim, index)
    _need(positions, "positions", torch.int64, (rows,), index)
    width = block_table.shape[-1] if isinstance(block_table, torch.Tensor) and block_table.dim() else 0
    _need(block_table, "block_table", torch.int32, (rows, width), index, True)
    dev = q.device
    out = torch.empty(rows, q_heads * head_dim, dtype=dtype, device=dev)
    # scratch of this call alone: from the caching allocator, so that calls on other streams and other captured graphs have theirs
    need = _attention_scratch.get((index, q_heads, kv_heads, head_dim))
    if need is None:
        with torch.cuda.device(index):
            need = max(_lib.load().bsb_paged_attention_scratch_bytes(rows, q_heads, kv_heads, head_dim), 16)
        _attention_scratch[(index, q_heads, kv_heads, head_dim)] = need
    scratch = torch.empty(need, dtype=torch.uint8, device=dev)
    _launch("bsb_paged_decode_attention", index, q.data_ptr(), k.data_ptr(), v.data_ptr(), _row_stride(q), _row_stride(k), _row_stride(v),
            cos.data_ptr(), sin.data_ptr(), cos.shape[0], positions.data_ptr(), block_table.data_ptr(), _row_stride(block_table), width,
            k_pages.data_ptr(), v_pages.data_ptr(), n, ks, vs, out.data_ptr(), rows, q_heads, kv_heads, head_dim, ps, _DTYPES[dtype],
            scratch.data_ptr(), need)
    return out


_attention_scratch = {}   # (device, head layout) -> bytes of scratch that one call needs, whatever its batch


def sample_step(logits, uniforms, tokens, temperature=None, top_k=None, top_p=None, min_p=None, pos=None, logprobs=None):
    """tokens[b] (int64 [batch]) drawn from softmax(logits[b] / temperature[b]) with the given uniform number uniforms[b]
    (fp32 [batch], in [0, 1)), after top-k, top-p and min-p (fp32 [batch], top_k int32 [batch]; None = off); then
    pos[0] += 1 (skipped when pos is None).  logits: [batch, vocab] fp16, bf16 or fp32 with unit inner stride.
    temperature 0: the first maximum, as `greedy_step`.  `logprobs` (fp32 [batch], optional) receives the log of the
    token's probability among those kept."""
    dtype = logits.dtype if isinstance(logits, torch.Tensor) else None
    if dtype not in _DTYPES:
        raise ValueError(f"logits must be fp16, bf16 or fp32, got {dtype}")
    index = _index(logits, "logits")
    _need(logits, "logits", dtype, (None, None), index, True)
    batch, vocab = logits.shape
    row = (batch,)
    _need(uniforms, "uniforms", torch.float32, row, index)
    _need(tokens, "tokens", torch.int64, row, index)
    if temperature is not None:
        _need(temperature, "temperature", torch.float32, row, index)
    if top_k is not None:
        _need(top_k, "top_k", torch.int32, row, index)
    if top_p is not None:
        _need(top_p, "top_p", torch.float32, row, index)
    if min_p is not None:
        _need(min_p, "min_p", torch.float32, row, index)
    if logprobs is not None:
        _need(logprobs, "logprobs", torch.float32, row, index)
    if pos is not None:
        _need(pos, "pos", torch.int64, (1,), index)
    _launch("bsb_sample_step", index, logits.data_ptr(), batch, vocab, _row_stride(logits), _DTYPES[dtype], uniforms.data_ptr(),
            None if temperature is None else temperature.data_ptr(), None if top_k is None else top_k.data_ptr(),
            None if top_p is None else top_p.data_ptr(), None if min_p is None else min_p.data_ptr(), tokens.data_ptr(),
            None if pos is None else pos.data_ptr(), None if logprobs is None else logprobs.data_ptr())
    return tokens
