"""The C library builds and the package imports without the Python extension, which says how to build it where it is needed."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def dry_run(*args):
    p = subprocess.run(["make", "-n", "-B", "-C", os.path.join(ROOT, "pcp_amd", "csrc"), *args], capture_output=True, text=True)
    return p.returncode, p.stdout, p.stderr


def test_library_needs_no_python():
    rc, out, err = dry_run("PYTHON=false")
    assert rc == 0 and "libpcp_grpo.so" in out and "tensor_lists.cpp" not in out and "torch" not in out + err, err


def test_extension_is_a_target_of_its_own():
    rc, out, _ = dry_run(f"PYTHON={sys.executable}", "python")
    assert rc == 0 and "tensor_lists.cpp" in out and "hipcc" not in out


PROGRAM = """
import sys
sys.modules["pcp_amd._tensors"] = None      # as where it has not been built
import torch
from pcp_amd import distill, grpo, scores, step
assert callable(step.pack_rollouts) and callable(step.sample_tokens) and callable(step.verify_drafts)
x = torch.zeros(8)
assert callable(scores.token_scores) and callable(distill.top_logits) and callable(grpo.grpo_loss_fwd_bwd)
for call in (lambda: step.grad_norm([x]), lambda: step.nesterov_update_many([x], [x], [x])):
    try:
        call()
    except ImportError as e:
        assert "make -C pcp_amd/csrc python" in str(e), e
    else:
        raise AssertionError("no error")
"""


def test_package_imports_without_the_extension():
    p = subprocess.run([sys.executable, "-c", PROGRAM], cwd=ROOT, capture_output=True, text=True)
    assert p.returncode == 0, p.stderr
