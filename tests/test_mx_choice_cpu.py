"""Which kernel a product with MXFP4 weights takes (mx_choice.h compiled for the host): the sizes of the GPU tests reach
every kernel, so that a change of the rules does not leave one untested."""
import ctypes
import os
import random
import subprocess

import pytest

import mx_sizes as S

HERE = os.path.dirname(os.path.abspath(__file__))
CLANG = "/opt/rocm/llvm/bin/clang++"
TYPES = {"f32": (1, 4), "f16": (4, 2), "bf16": (6, 2), "e4m3": (29, 1)}  # dtype code, bytes


@pytest.fixture(scope="module")
def choice(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("mx") / "mx_choice.so")
    subprocess.run([CLANG, "-x", "hip", "--offload-host-only", "--rocm-path=/opt/rocm", "-std=c++17", "-O1", "-shared",
                    "-fPIC", "-I", os.path.join(HERE, "..", "ptwm_amd", "csrc"),
                    os.path.join(HERE, "host", "mx_choice.hip"), "-o", so], check=True)
    lib = ctypes.CDLL(so)
    u32, u64 = ctypes.c_uint32, ctypes.c_uint64
    lib.mx_choice.argtypes = [u32, u64, u32, u32, u64, u64, u64, u64, u64, u64, ctypes.POINTER(u32)]

    def call(kind, tokens, rows, cols, x=0, x_stride=None, xs_stride=None, w=0, w_stride=None, s_stride=None):
        out = (u32 * 7)()
        lib.mx_choice(TYPES[kind][0], tokens, rows, cols, 4096 + x, cols if x_stride is None else x_stride,
                      cols // 32 if xs_stride is None else xs_stride, 4096 + w,
                      cols // 2 if w_stride is None else w_stride, cols // 32 if s_stride is None else s_stride, out)
        k = list(out)
        name = (S.SMALL,) if k[0] == 0 else S.few(k[1]) if k[0] == 1 else S.tile(*k[2:6])
        return name, bool(k[6])

    return call


@pytest.mark.parametrize("kind", TYPES)
def test_sizes_reach_their_kernels(choice, kind):
    for (tokens, rows, cols), want in S.SIZES[kind].items():
        got, aligned = choice(kind, tokens, rows, cols)
        assert got == want, (tokens, rows, cols)
        assert aligned == (want[0] == S.TILES)


@pytest.mark.parametrize("kind", TYPES)
def test_every_kernel_is_among_the_sizes(choice, kind):
    rng = random.Random(5)
    known = set(S.SIZES[kind].values())
    seen = set()
    for _ in range(20000):
        tokens = int(2 ** rng.uniform(0, 12))
        rows, cols = int(2 ** rng.uniform(0, 15)), 32 * int(2 ** rng.uniform(0, 9))
        name = choice(kind, tokens, rows, cols)[0]
        assert name in known, (tokens, rows, cols)
        seen.add(name)
    assert seen == known


@pytest.mark.parametrize("kind", TYPES)
def test_alignment(choice, kind):
    """Operands that no load of 16 bytes fits take the kernel's other form, and no other kernel."""
    size = TYPES[kind][1]
    for (tokens, rows, cols), want in S.SIZES[kind].items():
        if want[0] != S.TILES:
            continue
        for kw in (dict(w=2), dict(w_stride=cols // 2 + 8)):
            assert choice(kind, tokens, rows, cols, **kw) == (want, False)
        assert choice(kind, tokens, rows, cols, w_stride=cols // 2 + 16, x_stride=cols + 16 // size) == (want, True)
        split = kind == "f32" and want[3] == 4  # such tiles take x through registers in any case
        for kw in (dict(x=size), dict(x_stride=cols + 1)):
            still = split or (tokens == 1 and "x_stride" in kw)
            assert choice(kind, tokens, rows, cols, **kw) == (want, still)


@pytest.mark.parametrize("kind", TYPES)
def test_strides(choice, kind):
    """The stride of a single row changes nothing; others do where a tile's rows pass 32-bit offsets."""
    size = TYPES[kind][1]
    huge = 1 << 40
    for (tokens, rows, cols), want in S.SIZES[kind].items():
        if tokens == 1:
            one = choice(kind, tokens, rows, cols)
            assert one[0] == want and choice(kind, tokens, rows, cols, x_stride=huge + 1, xs_stride=huge + 1) == one
        assert choice(kind, tokens, rows, cols, x_stride=1 << 24, xs_stride=1 << 24, w_stride=1 << 24)[0] == want
    one = choice(kind, 70, 1, 4096)
    assert one[0][0] == S.TILES and choice(kind, 70, 1, 4096, w_stride=huge + 1, s_stride=huge + 1) == one
    want = choice(kind, *S.FAR)[0]
    assert want[:2] == (S.TILES, 32)
    for operand, key, n in (("x", "x_stride", size), ("x_scales", "xs_stride", 1), ("weight", "w_stride", 1),
                            ("scales", "s_stride", 1)):
        if operand == "x_scales" and kind != "e4m3":
            continue
        last = S.far_stride(operand, n)
        assert choice(kind, *S.FAR, **{key: last})[0] == want
        assert choice(kind, *S.FAR, **{key: last + 1})[0] == (S.SMALL,)
