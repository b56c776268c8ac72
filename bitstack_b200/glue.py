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
# Argument checks, outputs and scratch are in csrc/serving_torch.cpp: at small sizes these calls are a few microseconds of
# GPU work, and the same steps take longer than that in Python.

def page_tables(lens, new_tokens, block_table, free_pages, free_count, page_size: int, max_tokens: int = 0, lens_out=None, free_count_out=None):
    """One step of a paged cache's bookkeeping on the device: request b holds lens[b] tokens (int32 [batch]) and gets
    new_tokens[b] more; pages it lacks are popped from the stack free_pages[:free_count] and entered in its row of
    block_table (int32 [batch, width], updated in place).  lens and free_count (int32 [1]) are updated in place unless
    lens_out / free_count_out receive the new values.  A request whose row is too narrow, or for which the stack runs out
    (requests in order), is refused: it keeps its length.

    Returns (slots, positions, offsets, last): slot and position of every new token, request after request, int64
    [max_tokens], -1 for tokens of refused requests and behind the end; int32 [batch + 1] first token of every request;
    int64 [batch] position of the request's last new token, -1 when it has none or was refused."""
    return _lib.serving().page_tables(lens, new_tokens, block_table, free_pages, free_count, page_size, max_tokens, lens_out, free_count_out)


def release_pages(done, lens, block_table, free_pages, free_count, page_size: int) -> None:
    """Requests with done[b] (bool [batch]) give their pages back to the stack, and their length becomes 0 (in place).  A page
    that several rows list goes back once for each of them: rows that share pages are released with their own pages alone."""
    _lib.serving().release_pages(done, lens, block_table, free_pages, free_count, page_size)


def rope_paged_cache(q, k, v, cos, sin, positions, slots, k_pages, v_pages, q_heads, kv_heads, head_dim):
    """Rotary embedding of a batch of tokens (a prompt, or several requests' tokens) at `positions` (int64 [tokens]); k and v
    go to `slots` (int64 [tokens]) of k_pages / v_pages [num_pages, kv_heads, page_size, head_dim].  Returns the rotated q
    [tokens, q_heads * head_dim].  Position -1: padding (its q row is 0, nothing is cached); slot -1: not cached."""
    return _lib.serving().rope_paged_cache(q, k, v, cos, sin, positions, slots, k_pages, v_pages, q_heads, kv_heads, head_dim)


def paged_decode_attention(q, k, v, cos, sin, positions, block_table, k_pages, v_pages, q_heads, kv_heads, head_dim):
    """One new token per request at positions[b] (int64 [batch]; -1: idle row): rotary embedding of q and k, k and v written
    into the request's page (block_table int32 [batch, width]), then grouped-query attention over positions 0 .. positions[b].
    q, k, v: [batch, heads * head_dim], rows may be strided views; fp16 or bf16.  Returns [batch, q_heads * head_dim]."""
    return _lib.serving().paged_decode_attention(q, k, v, cos, sin, positions, block_table, k_pages, v_pages, q_heads, kv_heads, head_dim)


def sample_step(logits, uniforms, tokens, temperature=None, top_k=None, top_p=None, min_p=None, pos=None, logprobs=None):
    """tokens[b] (int64 [batch]) drawn from softmax(logits[b] / temperature[b]) with the given uniform number uniforms[b]
    (fp32 [batch], in [0, 1)), after top-k, top-p and min-p (fp32 [batch], top_k int32 [batch]; None = off); then
    pos[0] += 1 (skipped when pos is None).  logits: [batch, vocab] fp16, bf16 or fp32 with unit inner stride.
    temperature 0: the first maximum, as `greedy_step`.  `logprobs` (fp32 [batch], optional) receives the log of the
    token's probability among those kept."""
    _lib.serving().sample_step(logits, uniforms, tokens, temperature, top_k, top_p, min_p, pos, logprobs)
    return tokens
