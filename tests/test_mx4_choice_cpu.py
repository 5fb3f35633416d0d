"""Which kernel a product of two MXFP4 matrices takes (mx_choice.h compiled for the host): the sizes of the GPU tests
reach every kernel, so that a change of the rules does not leave one untested."""
import ctypes
import os
import random
import subprocess

import pytest

import mx4_sizes as S

HERE = os.path.dirname(os.path.abspath(__file__))
CLANG = "/opt/rocm/llvm/bin/clang++"


@pytest.fixture(scope="module")
def choice(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("mx4") / "mx4_choice.so")
    subprocess.run([CLANG, "-x", "hip", "--offload-host-only", "--rocm-path=/opt/rocm", "-std=c++17", "-O1", "-shared",
                    "-fPIC", "-I", os.path.join(HERE, "..", "ptwm_amd", "csrc"),
                    os.path.join(HERE, "host", "mx4_choice.hip"), "-o", so], check=True)
    lib = ctypes.CDLL(so)
    lib.mx4_choice.argtypes = [ctypes.c_uint64, ctypes.c_uint32, ctypes.c_uint32, ctypes.POINTER(ctypes.c_uint64),
                               ctypes.POINTER(ctypes.c_uint32)]

    def call(tokens, rows, cols, **kw):
        at = dict(x=4096, x_stride=cols // 2, xs=4096, xs_stride=cols // 32, w=4096, w_stride=cols // 2, s=4096,
                  s_stride=cols // 32)
        assert set(kw) <= set(at)
        out = (ctypes.c_uint32 * 2)()
        lib.mx4_choice(tokens, rows, cols, (ctypes.c_uint64 * 8)(*{**at, **kw}.values()), out)
        return S.KERNELS[out[0]], out[1]

    return call


def test_sizes_reach_their_kernels(choice):
    for (tokens, rows, cols), want in S.SIZES.items():
        dma = 0 if want == "small" else 2 if cols % 512 == 0 else 1
        assert choice(tokens, rows, cols) == (want, dma), (tokens, rows, cols)


def test_every_kernel_and_way_is_among_the_sizes(choice):
    known = {choice(*size) for size in S.SIZES}
    rng, seen = random.Random(6), set()
    for _ in range(20000):
        seen.add(choice(int(2 ** rng.uniform(0, 12)), int(2 ** rng.uniform(0, 15)), 32 * int(2 ** rng.uniform(0, 9))))
    assert {k for k, _ in seen} == set(S.KERNELS) == {k for k, _ in known}
    for kernel in set(S.KERNELS) - {"small"}:
        assert {(kernel, 1), (kernel, 2)} <= known


def test_alignment(choice):
    """Operands at other places take the kernel's other forms, and no other kernel."""
    for (tokens, rows, cols), want in S.SIZES.items():
        if want == "small":
            continue
        for kw in (dict(w=4097), dict(x=4104), dict(w_stride=cols // 2 + 8)):
            assert choice(tokens, rows, cols, **kw) == (want, 0)
        if tokens > 1:
            assert choice(tokens, rows, cols, x_stride=cols // 2 + 1) == (want, 0)
            assert choice(tokens, rows, cols, xs_stride=cols // 32 + 1) == (want, 1)
        for kw in (dict(s=4100), dict(xs=4097), dict(s_stride=cols // 32 + 8)):
            assert choice(tokens, rows, cols, **kw) == (want, 1)
        # scales past a row's last whole quad are not read, padded or not
        assert choice(tokens, rows, cols, s_stride=4096, xs_stride=4096)[1] == (2 if cols % 512 == 0 else 1)


def test_strides(choice):
    """A single row's stride is of no account; others are where a tile's rows pass 32-bit offsets."""
    odd = (1 << 40) + 1
    assert choice(1, 4096, 5120, x_stride=odd, xs_stride=odd) == ("32x32 by 8", 2)
    assert choice(70, 1, 4096, w_stride=odd, s_stride=odd) == ("32x32 by 8", 2)
    tokens, rows, cols = 40, 3000, 2208
    last = (2**32 - 1 - cols // 2) // 31
    for key in ("w_stride", "x_stride"):
        assert choice(tokens, rows, cols, **{key: last})[0] == "32x32 by 8"
        assert choice(tokens, rows, cols, **{key: last + 1})[0] == "small"
    assert choice(tokens, rows, cols, s_stride=odd, xs_stride=odd)[0] == "32x32 by 8"  # 64-bit addresses
