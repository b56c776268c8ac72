"""The decode kernel's passes over a larger batch follow each other closely: the next pass's operand preparation runs
beside the tail of this one.  Repeated calls on the same input must give the same bits, and every row what it gives alone."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [5, 16])
def test_back_to_back_passes_are_bit_identical(rows):
    from bitstack_b200.layer_bench import synthetic_projection
    dev = torch.device("cuda:0")
    mod = synthetic_projection(4096, 4096, 8, 10, dev, seed=91)
    x = torch.randn(rows, 4096, device=dev, generator=torch.Generator(device=dev).manual_seed(rows)).half()
    torch.cuda.synchronize()
    alone = []
    for lo in range(0, rows, 2):              # one pass at a time, nothing behind it
        alone.append(mod(x[lo:lo + 2]))
        torch.cuda.synchronize()
    alone = torch.cat(alone)
    got = [mod(x) for _ in range(40)]
    torch.cuda.synchronize()
    assert sum(not torch.equal(y, alone) for y in got) == 0
