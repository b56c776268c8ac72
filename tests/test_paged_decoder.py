"""The serving operators together, as a decoder runs them: ragged prompts, one step of all requests, sampling, requests
that come and go, a captured step."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model():
    from bitstack_b200 import decode
    shape = decode.LlamaShape("tiny", 2, 512, 4, 2, 1024, vocab=1000)
    return decode.BitStackLlamaDecoder(shape, decode.seeded_block_counts(shape, seed=3, lo=2, hi=4), "cuda:0", seed=5, max_len=128)


def _prompts(lengths, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 1000, (n,), generator=g) for n in lengths]


def _dense(model, prompt, tokens):
    """Logits of the dense decoder after the prompt and after each of `tokens`, one request alone."""
    model.prefill(prompt.to(model.device).view(1, -1))
    out = []
    for t in tokens:
        model.tokens.fill_(t)
        out.append(model._decode_fused().float()[0].clone())
        model.pos.add_(1)
    return out


@pytest.mark.parametrize("page_size", [1, 16, 24])
def test_ragged_requests_match_the_dense_decoder(model, page_size):
    """Every request's logits, step by step, against the dense decoder on that request alone (both are sums of fp16 products
    in another order: 2e-2 of the largest logit, as the fused dense step is held to)."""
    from bitstack_b200.serving import PagedDecoder
    prompts = _prompts([9, 1, 33, 16], seed=1)
    d = PagedDecoder(model, rows=5, num_pages=-(-512 // page_size), page_size=page_size)
    rows = d.submit(prompts)
    assert rows == [0, 1, 2, 3] and d.lens.tolist() == [9, 1, 33, 16, 0]
    fed, seen = [], []
    for _ in range(4):
        fed.append(d.tokens.clone())
        d.step()
        seen.append(d.logits.float().clone())
        assert d.positions.tolist()[4] == -1
    assert d.lens.tolist() == [13, 5, 37, 20, 0]
    for r, p in enumerate(prompts):
        for a, b in zip(_dense(model, p, [int(t[r]) for t in fed]), seen):
            assert (a - b[r]).abs().max() <= 2e-2 * a.abs().max()
    assert d.tokens[:4].tolist() == seen[-1][:4].argmax(-1).tolist()          # temperature 0


def test_captured_step_equals_the_eager_one_while_requests_come_and_go(model):
    """The same requests, numbers and settings, eagerly and through a captured graph: the same tokens and log-probabilities,
    bit for bit; pages of a released request serve the next one."""
    from bitstack_b200.serving import PagedDecoder
    runs = []
    for captured in (False, True):
        g = torch.Generator().manual_seed(7)
        d = PagedDecoder(model, rows=3, num_pages=12, page_size=8)
        if captured:
            d.capture()
            assert d.lens.tolist() == [0, 0, 0] and int(d.free_count) == 12
        seen = []
        a = d.submit(_prompts([5], 1), temperature=0.9, top_p=0.9, uniforms=torch.rand(1, generator=g))
        for _ in range(3):
            seen.append(d.step(torch.rand(3, generator=g)).tolist() + d.logprobs.tolist())
        b = d.submit(_prompts([20, 7], 2), temperature=1.2, top_k=20, min_p=0.02, uniforms=torch.rand(2, generator=g))
        for _ in range(4):
            seen.append(d.step(torch.rand(3, generator=g)).tolist() + d.logprobs.tolist())
        free = int(d.free_count)
        d.release(a)
        assert int(d.free_count) == free + 2 and d.free_rows() == a
        c = d.submit(_prompts([30], 3), temperature=0.7, uniforms=torch.rand(1, generator=g))
        assert c == a
        for _ in range(5):
            seen.append(d.step(torch.rand(3, generator=g)).tolist() + d.logprobs.tolist())
        d.release(b + c)
        assert int(d.free_count) == 12 and sorted(d.free_pages.tolist()) == list(range(12))
        runs.append(seen)
    assert runs[0] == runs[1]


def test_two_captured_steps_side_by_side(model):
    """Two decoders' graphs, replayed at the same time on two streams: neither disturbs the other's scratch.  (The projections
    share a workspace per stream, so each graph is captured, and replayed, on a stream of its own.)"""
    from bitstack_b200 import glue
    dev, outs, work = model.device, [], []
    for seed in range(2):
        g = torch.Generator(device=dev).manual_seed(seed)
        q, k, v = (torch.randn(6, h * 128, device=dev, generator=g).half() for h in (8, 2, 2))
        kp, vp = (torch.randn(200, 2, 16, 128, device=dev, generator=g).half() for _ in range(2))
        table = torch.randperm(200, device=dev, generator=g)[:6 * 33].int().view(6, 33)
        pos = torch.tensor([500, 17, -1, 511, 300, 3], device=dev)
        logits = torch.randn(6, 5000, device=dev, generator=g).half()
        u, tok = torch.rand(6, device=dev, generator=g), torch.zeros(6, dtype=torch.int64, device=dev)
        cos, sin = torch.rand(600, 128, device=dev, generator=g).half(), torch.rand(600, 128, device=dev, generator=g).half()
        p = torch.full((6,), 0.8, device=dev)

        def run(q=q, k=k, v=v, kp=kp, vp=vp, table=table, pos=pos, logits=logits, u=u, tok=tok, cos=cos, sin=sin, p=p):
            return glue.paged_decode_attention(q, k, v, cos, sin, pos, table, kp, vp, 8, 2, 128), glue.sample_step(logits, u, tok, top_p=p)
        want = [t.clone() for t in run()]
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            got = run()
        work.append((graph, stream, got, run))   # (the graph holds its inputs' addresses, `run` the inputs)
        outs.append(want)
    for _ in range(50):
        for graph, stream, _, _ in work:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for (_, _, got, _), want in zip(work, outs):
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_pool_exhaustion(model):
    from bitstack_b200.serving import OutOfPages, PagedDecoder
    d = PagedDecoder(model, rows=3, num_pages=4, page_size=8)
    with pytest.raises(OutOfPages):
        d.submit(_prompts([40], 1))
    assert int(d.free_count) == 4 and d.lens.tolist() == [0, 0, 0] and d.free_rows() == [0, 1, 2]
    d.submit(_prompts([16, 14], 1))                          # all four pages
    before = d.tokens.tolist()
    d.step()                                                 # row 0 needs a fifth page, row 1 has room for two more tokens
    assert d.positions.tolist() == [-1, 14, -1] and d.lens.tolist() == [16, 15, 0] and d.tokens.tolist()[0] == before[0]
    d.step()
    d.step()
    assert d.positions.tolist() == [-1, -1, -1] and d.lens.tolist() == [16, 16, 0]
    d.release([1])
    d.step()
    assert d.positions.tolist() == [16, -1, -1] and d.lens.tolist() == [17, 0, 0]
    with pytest.raises(ValueError):
        d.release([1])
    with pytest.raises(ValueError):
        d.submit([torch.zeros(0, dtype=torch.long)])
    with pytest.raises(ValueError):
        d.submit(_prompts([d.max_positions + 1], 1))


def test_prompts_outside_the_vocabulary_are_refused(model):
    from bitstack_b200.serving import PagedDecoder
    d = PagedDecoder(model, rows=2, num_pages=8, page_size=8)
    for bad in (torch.tensor([5, 1000]), torch.tensor([-1]), torch.tensor([1.0, 2.0])):
        with pytest.raises(ValueError):
            d.submit([torch.tensor([1, 2, 3]).to(bad.dtype), bad])
    assert int(d.free_count) == 8 and d.lens.tolist() == [0, 0] and d.free_rows() == [0, 1]
    d.release([])                                            # nobody ends
    assert d.submit([torch.tensor([999], dtype=torch.int32)]) == [0]


def test_a_request_up_to_its_last_position(model):
    """128 positions in pages of 24: six whole pages, 144 positions; then the row makes no step, and nothing is NaN."""
    from bitstack_b200 import _lib
    from bitstack_b200.serving import PagedDecoder
    d = PagedDecoder(model, rows=1, num_pages=8, page_size=24)
    assert d.max_positions == 144
    d.submit(_prompts([126], 1))
    for n in range(126, 146):
        d.step()
        assert torch.isfinite(d.logits).all()
        assert d.positions.tolist() == [n if n < 144 else -1]
    _lib.check_device_status()
    # the positions that the decoder's own tables hold are turned by the same numbers
    assert torch.equal(d.cos[:128], model.cos) and torch.equal(d.sin[:128], model.sin)


def test_a_prompt_that_fails_gives_its_pages_back(model, monkeypatch):
    from bitstack_b200.serving import PagedDecoder
    d = PagedDecoder(model, rows=2, num_pages=8, page_size=8)
    monkeypatch.setattr(PagedDecoder, "_prompt", lambda self, *a: (_ for _ in ()).throw(RuntimeError("no")))
    with pytest.raises(RuntimeError, match="no"):
        d.submit(_prompts([20], 1))
    assert int(d.free_count) == 8 and d.lens.tolist() == [0, 0] and d.free_rows() == [0, 1]


def test_generate(model):
    from bitstack_b200.serving import PagedDecoder
    d = PagedDecoder(model, rows=2, num_pages=64, page_size=4)
    a = d.generate(_prompts([7, 12], 4), steps=6)
    assert [len(x) for x in a] == [6, 6] and a == d.generate(_prompts([7, 12], 4), steps=6)
    assert int(d.free_count) == 64
    one = torch.tensor([7, 12, 3])
    assert d.generate([one], steps=3) == [d.generate([one, one], steps=3)[1]]
