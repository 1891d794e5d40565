"""Importing the package, under either name, neither needs nor loads torch: the calls that
take tensors load it themselves."""
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


def _python(code):
    return subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)


@pytest.mark.parametrize("name", ["rdnattention", "rdnattention_b200"])
def test_import_without_torch(name):
    res = _python(f"import sys; sys.modules['torch'] = None\nfrom {name} import *\n"
                  "print(callable(paged_kv_append), callable(flash_attn_paged), callable(paged_kv_accept),"
                  " len(SUPPORTED_HEAD_DIMS_PAGED), callable(flash_attn))")
    assert res.returncode == 0, res.stderr
    assert res.stdout.split() == ["True", "True", "True", "8", "True"]


@pytest.mark.parametrize("name", ["rdnattention", "rdnattention_b200"])
def test_import_leaves_torch_unloaded(name):
    res = _python(f"import sys\nimport {name}\n{name}.flash_attn_paged, {name}.__all__\nprint('torch' in sys.modules)")
    assert res.returncode == 0, res.stderr
    assert res.stdout.strip() == "False"


def test_first_paged_call_loads_torch():
    """A call that is refused, in a process that never imported torch itself."""
    res = _python("import rdnattention as R\n"
                  "try:\n    R.paged_kv_accept(None, None, None, None, None)\n"
                  "except TypeError as e:\n    print(e)")
    assert res.returncode == 0, res.stderr
    assert "must be torch.Tensors" in res.stdout
