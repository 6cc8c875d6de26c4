"""The compiled torch binding of the norm, the sort and the 4-bit products: what
it refuses because it goes past torch's dispatcher, and the package where it is
missing or was built against another torch."""

import importlib.util
import subprocess
import sys
from pathlib import Path

import pytest
import torch
import torch.autograd.forward_ad as fwd

from tests.conftest import ROOT

DEV = "cuda:0"


@pytest.mark.gpu
def test_forward_mode_derivatives_are_refused():
    """They would be left out without a word."""
    from int8blockwisegemm_b200 import int4, norm, permute
    T, K, topk = 4, 64, 2
    x, w = torch.randn(T, K, device=DEV), torch.randn(K, device=DEV)
    y, tw = torch.randn(T * topk, K, device=DEV), torch.rand(T, topk, device=DEV)
    ids = torch.zeros(T, topk, dtype=torch.int32, device=DEV)
    inv = torch.arange(T * topk, dtype=torch.int32, device=DEV)
    eft = torch.tensor([0, T * topk], device=DEV)
    one = torch.ones(T, device=DEV)
    packed, scale = int4.quantize_weights_int4(torch.randn(1, 32, K, device=DEV), 32, torch.bfloat16)
    eo = torch.tensor([0, T], dtype=torch.int32, device=DEV)
    xb = x.bfloat16()
    calls = [  # the tensors of a call, each of them with a tangent in turn
        (lambda a, b: norm.rms_norm(a, b), (x, w)), (lambda a, b: norm.rms_norm(x, w, 1e-6, a), (x, w)),
        (lambda a, b: norm.rms_norm_quant_int8(a, b), (x, w)),
        (lambda a, b: norm.rms_norm_backward(a, x, b, one), (x, w)),
        (lambda a, b: norm.rms_norm_backward(x, a, b, one, None, x), (x, w)),
        (lambda a, b: permute.moe_permute_train(a, ids, 1), (x, w)),
        (lambda a, b: permute.moe_unpermute_train(a, b, inv, eft), (y, tw)),
        (lambda a, b: permute.moe_permute_backward(a, inv, eft, T, topk), (y, tw)),
        (lambda a, b: permute.moe_unpermute_backward(x, a, b, inv, eft), (y, tw)),
        (lambda a, b: int4.int4_grouped_mv(a, packed, b, eo, 32), (xb, scale))]
    for call, args in calls:
        want = call(*args)
        with fwd.dual_level():
            call(*args)
            refused = 0
            for i in range(2):
                dual = [fwd.make_dual(a, torch.ones_like(a)) if i == j else a for j, a in enumerate(args)]
                try:
                    call(*dual)
                except RuntimeError as e:
                    assert "forward-mode" in str(e)
                    refused += 1
            assert refused >= 1
        again = call(*args)
        want, again = (t if isinstance(t, tuple) else (t,) for t in (want, again))
        assert all(a is b or torch.equal(a, b) for a, b in zip(want, again))


def run_python(code):
    res = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=ROOT, timeout=300)
    assert res.returncode == 0, res.stdout + res.stderr
    return res.stdout


def test_the_package_works_without_the_binding():
    """What is bound by ctypes does not need it; its own operators say what is
    missing."""
    out = run_python("""
import sys
class Missing:
    def find_spec(self, name, path=None, target=None):
        if name.endswith("._torch_ops"):
            raise ImportError("no such file")
sys.meta_path.insert(0, Missing())
import torch
import int8blockwisegemm_b200 as pkg
from int8blockwisegemm_b200 import _lib
assert torch.ops.int8_hybrid_moe.moe_permute_unpermute_supported()
assert _lib.LIB.i8moe_route_workspace_size(1, 8) == 64
x = torch.zeros(2, 8)
i = torch.zeros(2, 1, dtype=torch.int32)
for call in (lambda: pkg.norm.rms_norm(x, x[0]), lambda: pkg.permute.moe_permute_train(x, i, 4),
             lambda: pkg.int4.int4_grouped_mv(x, x, x, i)):
    try:
        call()
    except RuntimeError as e:
        assert "no such file" in str(e) and "_build.py" in str(e), e
        print("refused")
""")
    assert out.count("refused") == 3


def test_a_binding_of_another_torch_is_not_used():
    out = run_python("""
import torch
version, torch.__version__ = torch.__version__, "1.2.3+cu0"
from int8blockwisegemm_b200 import _lib, norm
torch.__version__ = version
try:
    norm.rms_norm(torch.zeros(2, 8), torch.zeros(8))
except RuntimeError as e:
    assert "built against torch " + version.split("+")[0] in str(e) and "1.2.3" in str(e), e
    print("refused")
""")
    assert out.count("refused") == 1


def test_the_binding_is_rebuilt_for_another_torch(tmp_path, monkeypatch):
    spec = importlib.util.spec_from_file_location("_i8moe_build_test", ROOT / "int8blockwisegemm_b200" / "_build.py")
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    so = tmp_path / "_torch_ops.so"
    monkeypatch.setattr(build, "TORCH_OPS", so)
    monkeypatch.setattr(build, "TORCH_STAMP", tmp_path / "stamp", raising=False)
    built = []

    def compiler(cmd, **kw):
        Path(cmd[cmd.index("-o") + 1]).write_text("built")
        built.append(cmd)
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(build.subprocess, "run", compiler)
    build.build_torch_ops()
    build.build_torch_ops()
    assert len(built) == 1  # up to date
    monkeypatch.setattr(torch, "__version__", "9.9.9+cu999")
    build.build_torch_ops()
    build.build_torch_ops()
    assert len(built) == 2


def test_a_pre_release_is_the_version_of_its_headers():
    run_python("""
import torch
version, torch.__version__ = torch.__version__, torch.__version__.split("+")[0] + "a0+git0"
from int8blockwisegemm_b200 import _lib
torch.__version__ = version
assert hasattr(_lib.TORCH_OPS, "rms_norm")
""")
