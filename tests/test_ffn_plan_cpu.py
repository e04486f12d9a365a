"""The gated feed-forward block's launch plans, enumerated on the host with the code that the kernels
run: tests/_ffn_plan_check.cu compiled for the CPU side only."""
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
PKG = os.path.join(os.path.dirname(HERE), "mps-deform-conv_b200")


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("plan") / "check")
    nvcc = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "bin", "nvcc")
    r = subprocess.run([nvcc, "-O2", "-std=c++17", "--expt-relaxed-constexpr", "-gencode", "arch=compute_100a,code=sm_100a",
                        "-I", os.path.join(os.path.dirname(HERE), "include"), "-I", os.path.join(PKG, "csrc"),
                        os.path.join(HERE, "_ffn_plan_check.cu"), "-o", out], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
    return out


def test_cut_products_add_every_k_block_once(program):
    """Each K block of each cut tile lies in one piece, the reduction adds the slots that the workers
    wrote and no others, and no worker has more than an even share (to a K block)."""
    r = subprocess.run([program], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout


def test_partial_buffers_hold_the_cut_products_sums_and_no_more(program):
    """At sizes of the block's products; and no cut gives a worker as much as it has without one."""
    r = subprocess.run([program, "plans"], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout
