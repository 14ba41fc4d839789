"""The gated feed-forward block on a B200: what stands before a call in its stream."""
import ctypes
import os
import shutil
import subprocess

import pytest
import torch

from ltxattn import device_status, gated_ffn, gated_ffn_backward

pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(autouse=True)
def no_kernel_timeouts():
    yield
    assert device_status(clear=True) == 0, "a kernel wait timed out"


def make(seed, m, hidden, inner, out, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s, k=1.0: (torch.randn(s, generator=g, device="cuda") * k).bfloat16()
    return (n(m, hidden, k=scale), n(inner, hidden, k=hidden ** -0.5), n(inner, hidden, k=hidden ** -0.5),
            n(out, inner, k=inner ** -0.5), n(m, out))


@pytest.fixture(scope="module")
def stays_on(tmp_path_factory):
    lib = tmp_path_factory.mktemp("stays_on") / "stays_on.so"
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-O2", "-shared", "-Xcompiler", "-fPIC",
                    os.path.join(HERE, "c", "stays_on.cu"), "-o", str(lib)], check=True)
    return ctypes.CDLL(str(lib)).launch_stays_on


@pytest.mark.parametrize("m", [1, 60])
def test_a_call_behind_a_long_kernel(stays_on, m):
    # The kernel before lets the call's first kernel start at once and stays for 2.4 s, longer than a wait in a kernel
    # may take (2 s): those waits are for the kernel's own loads and products, and start when it may run.
    x, wg, wu, wd, dout = make(31, m, 256, 520, 264)
    y, gate, up = gated_ffn(x, wg, wu, wd, save=True)
    grads = gated_ffn_backward(x, wg, wu, wd, gate, up, dout)
    torch.cuda.synchronize()
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert stays_on(ctypes.c_uint32(2400), stream) == 0
    again = gated_ffn(x, wg, wu, wd, save=True)
    assert stays_on(ctypes.c_uint32(2400), stream) == 0
    grads_again = gated_ffn_backward(x, wg, wu, wd, gate, up, dout)
    torch.cuda.synchronize()
    assert device_status(clear=True) == 0
    assert all(torch.equal(a, b) for a, b in zip(again, (y, gate, up)))
    assert all(torch.equal(a, b) for a, b in zip(grads_again, grads))
