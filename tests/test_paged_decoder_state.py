"""PagedDecoder where a call fails or is out of the ordinary: the requests that run go on as if it had not been made."""
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


@pytest.mark.parametrize("captured_before", [False, True])
@pytest.mark.parametrize("failing", [1, 2, 3])                # two warm-up steps, then the captured one
def test_a_capture_that_fails_leaves_the_requests_running(model, monkeypatch, failing, captured_before):
    from bitstack_b200.serving import PagedDecoder
    runs = []
    for fails in (False, True):
        d = PagedDecoder(model, rows=3, num_pages=40, page_size=8)
        if captured_before:
            d.capture()
        d.submit(_prompts([11, 30], 1))
        d.step()
        before = [t.tolist() for t in (d.active, d.tokens, d.logprobs, d.positions, d.lens)]
        logits = d.logits.clone()
        if fails:
            calls, real = [], PagedDecoder._step

            def step(self):
                calls.append(1)
                if len(calls) == failing:
                    self.positions.fill_(-7)
                    raise RuntimeError("no")
                real(self)
            with monkeypatch.context() as m:
                m.setattr(PagedDecoder, "_step", step)
                graph = d._graph
                with pytest.raises(RuntimeError, match="no"):
                    d.capture()
            assert d._graph is graph and len(calls) == failing
            assert [t.tolist() for t in (d.active, d.tokens, d.logprobs, d.positions, d.lens)] == before
            assert torch.equal(d.logits, logits)
        runs.append([d.step().tolist() + d.positions.tolist() for _ in range(4)])
        d.capture()                                           # and a later one succeeds
        runs[-1] += [d.step().tolist() + d.positions.tolist() for _ in range(3)]
    assert runs[0] == runs[1] and all(r[3:5] == [11 + 1 + i, 30 + 1 + i] for i, r in enumerate(runs[0]))


def test_captured_steps_share_no_scratch(model, monkeypatch):
    """Two decoders whose captures meet the same stream handle (handles come from a small pool), and eager calls on it: each uses
    scratch of its own, so their replays may run side by side."""
    from bitstack_b200 import linear
    from bitstack_b200.serving import PagedDecoder
    stream, used, real = torch.cuda.Stream(), {}, linear.get_workspace

    def spy(device, nbytes):
        t = real(device, nbytes)
        used.setdefault(who + (" captured" if torch.cuda.is_current_stream_capturing() else " eager"), set()).add(t.data_ptr())
        return t
    monkeypatch.setattr(linear, "get_workspace", spy)
    monkeypatch.setattr(torch.cuda, "Stream", lambda *a, **k: stream)
    who = "before"
    decoders = []
    with torch.cuda.stream(stream):
        first = PagedDecoder(model, rows=3, num_pages=20, page_size=8)
        first.generate(_prompts([9, 5], 2), steps=3)
    stream.synchronize()
    for who in ("a", "b"):
        d = PagedDecoder(model, rows=3, num_pages=20, page_size=8)
        d.capture()
        decoders.append(d)
    who = "after"
    with torch.cuda.stream(stream):
        first.generate(_prompts([9, 5], 2), steps=3)
    stream.synchronize()
    a, b = used["a captured"], used["b captured"]
    assert a and b and not a & b and not (a | b) & (used["before eager"] | used["after eager"])
    assert used["before eager"] == used["after eager"]        # the calls outside keep theirs
    assert [{t.data_ptr() for t in d._graph.scratch} for d in decoders] == [a, b]
    runs = []
    for d in decoders:
        rows = d.submit(_prompts([9, 5], 2))
        runs.append([d.tokens[rows].tolist()] + [d.step()[rows].tolist() for _ in range(2)])
    assert runs[0] == runs[1] and [list(t) for t in zip(*runs[0])] == first.generate(_prompts([9, 5], 2), steps=3)
