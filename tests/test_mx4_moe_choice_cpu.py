"""How the products of a mixture-of-experts layer on MXFP4 experts are made (mx_choice.h compiled for the host): the
sizes of the GPU tests reach every way, so that a change of the rules does not leave one untested."""
import ctypes
import os
import random
import subprocess

import pytest

import mx4_moe_sizes as S

HERE = os.path.dirname(os.path.abspath(__file__))
CLANG = "/opt/rocm/llvm/bin/clang++"
TYPE = {"f32": 1, "f16": 4, "bf16": 6}


@pytest.fixture(scope="module")
def choice(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("mx4_moe") / "mx4_moe_choice.so")
    subprocess.run([CLANG, "-x", "hip", "--offload-host-only", "--rocm-path=/opt/rocm", "-std=c++17", "-O1", "-shared",
                    "-fPIC", "-I", os.path.join(HERE, "..", "ptwm_amd", "csrc"),
                    os.path.join(HERE, "host", "mx4_moe_choice.hip"), "-o", so], check=True)
    lib = ctypes.CDLL(so)

    def call(tokens, experts, top_k, cols, inner, kind, **kw):
        at = {}
        for name, rows, n in (("gate", inner, cols), ("up", inner, cols), ("down", cols, inner)):
            at |= {name: 4096, name + "_stride": n // 2, name + "_expert": rows * n // 2, name + "_scales_stride": n // 32}
        assert set(kw) <= set(at)
        out = (ctypes.c_uint32 * 7)()
        lib.mx4_moe_choice((ctypes.c_uint64 * 6)(tokens, experts, top_k, cols, inner, TYPE[kind]),
                           (ctypes.c_uint64 * 12)(*{**at, **kw}.values()), out)
        return dict(inner=S.INNER[out[0]], outer=S.OUTER[out[1]], inner_dma=bool(out[2]), outer_dma=bool(out[3]),
                    routed=bool(out[4]), span=out[5], chunks=out[6])

    return call


def test_sizes_reach_their_ways(choice):
    for size, want in S.SIZES.items():
        c = choice(*size)
        assert (c["inner"], c["outer"], c["routed"]) == want, (size, c)
        assert c["inner_dma"] and c["outer_dma"]


def test_every_way_is_among_the_sizes(choice):
    """Of the combinations that sizes of many magnitudes reach too, but for rare ones."""
    known = {tuple(choice(*s)[k] for k in ("inner", "outer")) for s in S.SIZES}
    rng, seen = random.Random(8), {}
    for _ in range(60000):
        experts = int(2 ** rng.uniform(0, 10.01))
        c = choice(int(2 ** rng.uniform(0, 6.01)), experts, min(experts, rng.randint(1, 32)), 32 * int(2 ** rng.uniform(0, 12)),
                   32 * int(2 ** rng.uniform(0, 12)), rng.choice(list(TYPE)))
        way = c["inner"], c["outer"]
        seen[way] = seen.get(way, 0) + 1
    assert {w[0] for w in seen} == set(S.INNER) == {w[0] for w in known}
    assert {w[1] for w in seen} == set(S.OUTER) == {w[1] for w in known}
    assert set(seen) <= known, set(seen) - known
    for routed in (False, True):
        assert {v[0] for v in S.SIZES.values() if v[2] == routed} >= {"64 rows", "stream 2", "stream 4"}


def test_alignment(choice):
    """Codes at other places go through registers, by the kernels that can."""
    ways = set()
    for size in S.SIZES:
        rows = ("16 rows", "64 rows")
        experts, cols, inner = size[1], size[3], size[4]
        for kw in (dict(gate=4097), dict(up=4104), dict(gate_stride=cols // 2 + 1), dict(up_expert=inner * cols // 2 + 8)):
            c = choice(*size, **kw)
            if "up_expert" in kw and experts == 1:
                continue
            assert c["inner"] in rows and not c["inner_dma"] and c["outer_dma"]
            ways.add(c["inner"])
        for kw in (dict(down=4097), dict(down_stride=inner // 2 + 4)):
            c = choice(*size, **kw)
            assert c["outer"] != "chunks" and not c["outer_dma"] and c["inner_dma"]
            ways.add(c["outer"])
    assert ways == {"16 rows", "64 rows", "sums of 1", "sums of 2"}


def test_strides(choice):
    """Columns in registers want gate and up alike, and 16 rows within 32-bit offsets."""
    size = (21, 6, 2, 2144, 3232, "f32")
    assert choice(*size, up_stride=2048)["inner"] == "64 rows"
    assert choice(*size, gate_scales_stride=68)["inner"] == "64 rows"
    for key in ("gate_stride", "up_scales_stride"):
        pair = {k: None for k in (key, key.replace("gate", "up") if "gate" in key else key.replace("up", "gate"))}
        assert choice(*size, **dict.fromkeys(pair, (1 << 27) - 16))["inner"] == "stream 2"
        assert choice(*size, **dict.fromkeys(pair, 1 << 27))["inner"] == "64 rows"
    for key in ("down_stride", "down_scales_stride"):
        assert choice(*size, **{key: (1 << 27) - 16})["outer"] == "chunks"
        assert choice(*size, **{key: 1 << 27})["outer"] == "64 rows"


def test_chunks(choice):
    """Chunks cover a row, each with a step for eight wavefronts at most."""
    for steps in range(1, 129):
        c = choice(64, 1, 1, 64, steps * 256, "bf16")
        if c["outer"] == "chunks":
            assert 1 <= c["span"] <= 8 and c["chunks"] <= 16
            assert (c["chunks"] - 1) * c["span"] < steps <= c["chunks"] * c["span"]
        else:
            assert steps <= 3 and c["chunks"] == 1
    assert choice(64, 1, 1, 64, 129 * 256, "bf16")["outer"] == "64 rows"
