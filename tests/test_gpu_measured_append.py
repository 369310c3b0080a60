"""The measured cases' plain form of the append has the scales that the library's has, and the same values come back, bit for bit."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "perf", "operators.py")


@pytest.mark.parametrize("dtype,requests,prompt,held", [("f32", 9, 2048, 1000), ("bf16", 48, 0, 8000), ("f16", 7, 100, 500)])
def test_same_bits(gpu, dtype, requests, prompt, held):
    torch = gpu
    spec = importlib.util.spec_from_file_location("measured_operators", PATH)
    ops = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ops)
    case = {"kind": "append", "dtype": dtype, "requests": requests, "prompt": prompt, "held": held, "page": 64, "kv_heads": 8,
            "head_dim": 128}
    out = []
    for own in (False, True):
        ops.own = own
        s = ops.prepare(case, 5)
        out.append([x.clone() for x in ops.run(s)])
    torch.cuda.synchronize()
    for name, x, y in zip(("key scales", "value scales", "keys", "values"), *out):
        assert torch.equal(x, y), f"{name}: {int((x != y).sum())} of {x.numel()} differ"
