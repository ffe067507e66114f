"""The package without the types of 4-bit caches, as a torch before 2.8 is: everything imports, other formats work as ever."""

from __future__ import annotations

import re
import subprocess
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1] / "prism-infer_amd"

WITHOUT = """
import importlib, pkgutil, sys
import torch
for name in ("float4_e2m1fn_x2", "float8_e8m0fnu"):
    delattr(torch, name)
sys.path.insert(0, sys.argv[1])
import prism_infer
for module in pkgutil.walk_packages(prism_infer.__path__, "prism_infer."):
    if not module.name.endswith(("_host_ops", "libprism_mi355x")):
        importlib.import_module(module.name)
from prism_infer import _native
from prism_infer.engine import kv_quantization as quant
from prism_infer.ops.kv_cache_store import is_fp4_cache_tensor, store_kvcache
from prism_infer.ops.paged_fp4 import is_fp4

fp8 = torch.float8_e4m3fn
x = torch.randn(3, 2, 64).bfloat16()
for scaled in (True, False):
    kc, vc = (torch.zeros(2, 16, 2, 64, dtype=fp8) for _ in range(2))
    scales = [torch.zeros(2, 16, 2) for _ in range(2)] if scaled else [None, None]
    store_kvcache(x, x, kc, vc, torch.tensor([0, 17, 5], dtype=torch.int32), *scales)
    held = kc.float() * (scales[0][..., None] if scaled else 1)
    assert (held.flatten(0, 1)[[0, 17, 5]] - x.float()).abs().max() < 0.3
assert not any(is_fp4_cache_tensor(t) or is_fp4(t) for t in (x, kc, kc.view(torch.uint8)))
bytes_ = quant.kv_block_storage_bytes(num_layers=1, page_size=16, num_kv_heads=2, head_dim=64, payload_dtype=fp8, token_head_scales=True)
assert (bytes_.payload, bytes_.scales) == (4096, 256)
assert _native.DTYPE_FP4_E2M1 not in _native._TORCH_TO_CODE.values()
print("done")
"""


def test_the_package_imports_and_stores_without_4bit_types():
    run = subprocess.run([sys.executable, "-c", WITHOUT, str(ROOT)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.split()[-1:] == ["done"], run.stderr


def test_the_host_path_names_4bit_types_only_where_they_may_be_missing():
    """Dependent names of a partial specialisation: a torch without them builds the file with types that no tensor has."""

    source = (ROOT / "csrc_host" / "host_ops.cpp").read_text()
    guard = re.search(r"template <typename T>\nstruct Fp4Types<T, std::void_t<.*?\n};\n", source, re.S)
    assert guard
    rest = source.replace(guard.group(), "")
    assert "Float4_e2m1fn_x2" not in rest and "Float8_e8m0fnu" not in rest
