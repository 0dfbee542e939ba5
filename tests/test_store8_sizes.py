"""nnhip_kv8_append of more heads of tokens than its kernel of rows can number: which launches a call makes, from its sizes
alone. Nothing is launched (launch_stub.c stands in for the runtime), so this runs without a GPU and the pointers are never
followed."""
import os
import shutil
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CHILD = """
import ctypes, sys
ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
sys.path[:0] = [{here!r}, {package!r}]
from chunk_helpers import Pages8, library
P, tokens, heads, q_heads, dim = 4096, *map(int, sys.argv[2:])
c = Pages8(P, 1 << 24, 1 << 25, 1 << 26, P, 1 << 20, 16, 1 << 20, 16, heads, dim, heads * dim)
f = heads * dim
q = (P, q_heads * dim, 1) if q_heads else (None, 0, 0)
print("status", library().nnhip_kv8_append(c, P, f, 1, P, f, 1, *q, *q, q_heads, tokens, P, P, None, None, 0, 0, None), flush=True)
"""


def divided(n, d):
    """n / d as FastDiv (kv_pages.hpp) forms it."""
    s = max(d - 1, 0).bit_length()
    return n * (((1 << (31 + s)) + d - 1) // d) >> (31 + s)


@pytest.fixture(scope="module")
def stub(tmp_path_factory):
    cc = shutil.which("gcc")
    if not cc:
        pytest.skip("no C compiler")
    so = str(tmp_path_factory.mktemp("stub") / "launch_stub.so")
    subprocess.run([cc, "-shared", "-fPIC", "-O1", "-o", so, os.path.join(HERE, "launch_stub.c")], check=True)
    return so


def launches(stub, *sizes):
    code = CHILD.format(here=HERE, package=os.path.join(os.path.dirname(HERE), "neuralnet.cpp_amd"))
    out = subprocess.run([sys.executable, "-c", code, stub, *map(str, sizes)], check=True, capture_output=True, text=True).stdout
    lines = [line.split() for line in out.splitlines()]
    assert ["status", "0"] in lines, out
    return [tuple(map(int, x[1:])) for x in lines if x[0] == "launch"]


def test_quotients_past_31_bits():
    assert divided(3020636529, 190) == 3020636529 // 190 + 1
    assert divided(3170893823, 189) == 3170893823 // 189 + 1
    for d in (3, 189, 190, 65535):
        for n in (2 ** 31 - 1, 2 ** 31 - d, 2 ** 31 // d * d, 2 ** 31 // d * d - 1):
            assert divided(n, d) == n // d


# tokens, key heads, query heads: 95 + 95 slots, 63 + 63 + 63, 64 + 64; the number of heads of tokens on either side of 2^31
@pytest.mark.parametrize("dim", [4, 8])
@pytest.mark.parametrize("tokens,heads,q_heads", [(15_900_000, 95, 0), (16_777_216, 63, 63), (1 << 24, 64, 0), ((1 << 24) - 1, 64, 0),
                                                  ((1 << 24) - 3, 64, 0), (11_300_000, 95, 0), (1000, 95, 0)])
def test_heads_of_tokens_are_numbered_in_31_bits(stub, tokens, heads, q_heads, dim):
    slots = 2 * heads + q_heads
    made = launches(stub, tokens, heads, q_heads, dim)
    assert len(made) == 1
    x, y, z, threads = made[0]
    assert threads == 256 and z == 1
    if y == 1:                 # a thread a head of a token
        assert tokens * slots <= x * threads <= 2 ** 31
    else:                      # a workgroup 32 tokens of a head
        assert (x, y) == (-(-tokens // 32), slots)
        assert tokens * slots > 2 ** 31 - 512
