"""A native library built before the operators of the 4-bit cache: the package imports, host tensors
are served, and a GPU call of a missing one says what to do."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# The schemas of such a library, in place of loading one.
SCRIPT = r"""
import torch

def load(path):
    lib = torch.library.Library("quant_ops", "DEF")
    lib.define("flatquant_dynamic_quantize(Tensor input, Tensor left_trans, Tensor right_trans, float clip_ratio=1, "
               "bool pack_int32=False) -> (Tensor, Tensor)")
    lib.define("int4_matmul(Tensor a, Tensor b, Tensor scale_a, Tensor scale_b) -> Tensor")
    lib.define("int4_matmul_ex(Tensor a, Tensor b, Tensor scale_a, Tensor scale_b, ScalarType? out_dtype=None) -> Tensor")
    lib.define("dequantize_int4(Tensor quantized, Tensor scales, bool packed_int32=False) -> Tensor")
    load.keep = lib

torch.ops.load_library = load
import quant_ops_amd as qo
from torch._subclasses.fake_tensor import FakeTensorMode

assert qo.CUDA_AVAILABLE
assert torch.ops.quant_ops.int4_matmul.default is not None
host = qo.kv4_cache(1, 16, 1, 64, device="cpu")
one = torch.ones(1, 1, 64)
qo.kv4_append(host, one, one, torch.zeros(1, dtype=torch.int64))      # host tensors need no library
assert bool((qo.kv4_read(host, torch.zeros(1, dtype=torch.int64))[0] == 1).all())
with FakeTensorMode():
    cache = qo.kv4_cache(2, 16, 1, 64)
    x = torch.empty(2, 1, 64, device="cuda")
    slots = torch.empty(2, dtype=torch.int64, device="cuda")
    table, n = torch.empty(2, 1, dtype=torch.int32, device="cuda"), torch.empty(2, dtype=torch.int32, device="cuda")
    for call in (lambda: qo.kv4_append(cache, x, x, slots), lambda: qo.kv4_read(cache, slots),
                 lambda: qo.kv4_attention(x, cache, table, n)):
        try:
            call()
        except RuntimeError as e:
            assert "rebuild" in str(e), e
        else:
            raise SystemExit("accepted")
import quant_ops_amd._build
print("ok")
"""


def test_package_imports():
    got = subprocess.run([sys.executable, "-c", SCRIPT], cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert got.returncode == 0 and got.stdout.strip().endswith("ok"), got.stderr[-2000:]
