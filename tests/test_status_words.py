"""Waits that gave up and indices outside their tensor are reported side by side: neither hides the other.

The wait runs out in the tuning build's mode for it (a barrier that nothing sets, time limit lowered to 20 ms: every role gives up
and the kernel returns normally); the bad index is a token list that is cut, which no kernel follows.  In a child process, so that
the tuning library and its status words stay out of the other tests."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHILD = r'''
import ctypes as C, os, sys
import numpy as np, torch
sys.path.insert(0, os.environ["BSB_ROOT"])
from oracle import bitstack_oracle as orc
from bitstack_b200 import _lib, glue, BitStackLinear
lib = _lib.load()
tuning = C.CDLL(_lib.LIB_PATH)
dev = torch.device("cuda:0")
m, n, nb = 640, 1024, 3
q, u, vt = orc.synthetic_layer(m, n, nb, seed=1)
mod = BitStackLinear(w_bit=nb, in_features=n, out_features=m, k=16, bias=False, no_avd=False, dev=dev, fused_level=10)
for j in range(nb):
    getattr(mod, f"qweight_{j}").copy_(torch.from_numpy(q[j]))
    getattr(mod, f"u_{j}").copy_(torch.from_numpy(u[j]))
    getattr(mod, f"vt_{j}").copy_(torch.from_numpy(vt[j]))
mod.stack_blocks()
x = torch.from_numpy(orc.synthetic_input(1, n, seed=2))
good = mod(x.to(dev))
hx, hy = x.contiguous(), torch.zeros(1, m, dtype=torch.float16)
dx, dy = torch.zeros(1, n, dtype=torch.float16, device=dev), torch.zeros(1, m, dtype=torch.float16, device=dev)
ws = torch.empty(64 << 20, dtype=torch.uint8, device=dev)
d = mod.weight_desc(dev)


def host_call():
    return lib.bsb_linear_forward_host(C.byref(d), hx.data_ptr(), 1, hy.data_ptr(), dx.data_ptr(), dy.data_ptr(), ws.data_ptr(), ws.numel(),
                                       _lib.ALGO_GEMV_TC5, torch.cuda.current_stream().cuda_stream)


def cut_list():                                         # 5 new tokens, a list of 2
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)
    glue.page_tables(i(0), i(5), torch.full((1, 4), -1, dtype=torch.int32, device=dev), i(1, 2, 3), i(3), 8, 2)


code = C.c_int32(0)
assert host_call() == 0 and torch.equal(hy, good.cpu())
cut_list()
torch.cuda.synchronize()
assert host_call() == 0 and torch.equal(hy, good.cpu()), "a bad index elsewhere is not this call's failure"
assert lib.bsb_set_wait_limit_ms(20) == 0
assert tuning.bsb_tuning_set_mode(3) == 0               # the Z' loader never loads
rc = host_call()
assert bool(torch.isnan(hy).all()) and rc == -5, (rc, "outputs are NaN: the call has to say so, whatever was pending")
assert tuning.bsb_tuning_set_mode(0) == 0
assert lib.bsb_read_status(C.byref(code), 0) == -5 and 0 < code.value < 61, code.value
try:
    _lib.check_device_status()
    raise SystemExit("the wait that gave up was not reported")
except _lib.BitStackDeviceTimeout:
    pass
assert lib.bsb_read_status(C.byref(code), 0) == -6 and code.value == 63, code.value
try:
    _lib.check_device_status()
    raise SystemExit("the index was not reported")
except _lib.BitStackDeviceIndexError:
    pass
assert lib.bsb_read_status(C.byref(code), 1) == 0 and code.value == 0
assert host_call() == 0 and torch.equal(hy, good.cpu())
print("BOTH_REPORTED", flush=True)
'''


@pytest.mark.gpu
def test_a_bad_index_does_not_hide_a_wait_that_gave_up():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from bitstack_b200 import build
    lib = build.TUNING_LIB
    if not os.path.exists(lib):
        lib = build.build_tuning()
    env = dict(os.environ, BITSTACK_B200_LIB=lib, BSB_ROOT=ROOT)
    out = subprocess.run([sys.executable, "-c", CHILD], env=env, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "BOTH_REPORTED" in out.stdout, out.stdout[-2000:] + out.stderr[-4000:]
