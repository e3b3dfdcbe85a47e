"""The paged-serving example end to end: lengths, and the last step against fp32 attention over the cache."""
import importlib.util
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def example():
    path = Path(__file__).resolve().parents[1] / "k-search_b200" / "examples" / "paged_serving.py"
    spec = importlib.util.spec_from_file_location("paged_serving", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


# One fp16 (bf16) rounding of the output is 2^-12 (2^-9) relative to each element; the weights' and the
# queries' roundings add a few of the same size.
@pytest.mark.parametrize("kw,tol", [
    (dict(requests=3, system=64, prompt=40, steps=20), 4 * 2 ** -12),
    (dict(requests=40, system=1024, prompt=90, steps=4, Hq=28, Hkv=4, page_size=32, dtype=torch.bfloat16), 4 * 2 ** -9),
    (dict(requests=5, system=0, prompt=33, steps=2, Hq=15, Hkv=5, D=64), 4 * 2 ** -12),
])
def test_paged_serving_example(kw, tol):
    r = example().run(quiet=True, **kw)
    assert r["lens"] and r["device_error"] == 0
    assert r["error"] < tol, r
