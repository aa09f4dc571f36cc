"""What the Python binding says of torch tensors that it cannot take.  In processes of their own: torch brings a HIP runtime along."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PYHOST = os.path.join(ROOT, "pocket-tts.cpp_amd", "pyhost")


def _run(body):
    code = f"import sys\nsys.path.insert(0, {PYHOST!r})\nimport ptts_lib, ptts_paged as P\n" + body + "\nprint('DONE')\n"
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "DONE" in r.stdout, r.stdout + r.stderr
    return r.stdout


GRAD = r'''
import torch
x, pos, freq = torch.zeros(5, 4, 64), torch.zeros(5, dtype=torch.int32), torch.zeros(32, dtype=torch.float64)
def said(f):
    try:
        f()
    except ptts_lib.PttsError as e:
        return str(e)
    raise AssertionError("not refused")
want = x.clone().requires_grad_()
for t in (want, want * 2, torch.nn.Parameter(x)):          # a leaf, a result, a parameter
    assert said(lambda: P.rotary_append(t, None, None, pos, freq)).startswith("q: requires gradients")
    with torch.no_grad():
        assert "not on the GPU" in said(lambda: P.rotary_append(t, None, None, pos, freq))
    with torch.inference_mode():
        assert "not on the GPU" in said(lambda: P.rotary_append(t, None, None, pos, freq))
    assert "not on the GPU" in said(lambda: P.rotary_append(t.detach(), None, None, pos, freq))
assert "not on the GPU" in said(lambda: P.rotary_append(x, None, None, pos, freq))
'''


def test_tensors_that_require_gradients_are_refused():
    _run(GRAD)


OLD = r'''
class Tensor:                        # what a torch without the table looks like from here
    def data_ptr(self):
        return 0
try:
    P.rotary_append(Tensor(), None, None, None, None)
except ptts_lib.PttsError as e:
    assert "Tensor publishes no exchange table" in str(e), e
else:
    raise AssertionError("not refused")
try:
    P.rotary_append([1.0], None, None, None, None)
except ptts_lib.PttsError as e:
    assert "a torch tensor on the GPU or a DeviceArray is required, got list" in str(e), e
else:
    raise AssertionError("not refused")
'''


def test_tensors_without_the_exchange_table_are_told_so():
    _run(OLD)
