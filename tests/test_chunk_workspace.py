"""What nnhip_attn_chunk and nnhip_attn_chunk8 ask for their ranges' results: bounded by the card's workgroups, however many
tokens the prompts have. Sizes alone: no GPU."""
import pytest

from chunk_helpers import Pages, Pages8, library

P = 4096
MIB = 1 << 20


def need(bits, batch, width, page, heads, dim, q_heads, tokens, most):
    sizes = (batch, width, batch * width, page, heads, dim, heads * dim)
    if bits == 8:
        return library().nnhip_attn_chunk8_workspace_bytes(Pages8(P, P, P, P, P, *sizes), q_heads, tokens, most)
    return library().nnhip_attn_chunk_workspace_bytes(Pages(P, P, P, *sizes), q_heads, tokens, most)


def parts(bits, batch, width, page, heads, dim, q_heads, tokens):
    """Most that the keys' and values' parts take: 32 positions a tile, each value of a key or value in two halves of two
    bytes (one of 8 bits), key and value dims in multiples of 16 and 32 from 32 on, two scales a position, 16 bytes more."""
    halves = 2 if bits == 32 else 1
    tile = 32 * 2 * halves * (max(-(-dim // 16), 2) * 16 + max(-(-dim // 32), 1) * 32) + 32 * 8 + 16
    one = -(-width * page // 32) * tile
    pieces = min(batch, tokens * (q_heads // heads) // 33 + 1) * heads
    return one * min(pieces, max(1, (2 << 30) // one))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("batch,each,heads,q_heads,dim", [
    (2, 8192, 8, 32, 128), (2, 8192, 1, 32, 128), (3, 5000, 2, 32, 128), (7, 3900, 16, 16, 80), (2, 500, 1, 32, 128),
    (2, 2000, 1, 16, 128), (1, 8192, 8, 32, 128), (64, 100, 8, 32, 128), (2, 60000, 1, 64, 128), (2, 40, 1, 1, 64), (600, 40, 1, 32, 128)])
def test_results_of_ranges(batch, each, heads, q_heads, dim, bits):
    """At most 8 workgroups a CU and another for every sequence and key head where these are fewer, of 32 rows each, and two
    workgroups a CU of 128 rows: (2 * 2048 * 32 + 512 * 128) results of dim + 2 floats, under 128 MiB."""
    page = 16
    width = -(-(each + 1000) // page)
    room = parts(bits, batch, width, page, heads, dim, q_heads, batch * each)
    got = need(bits, batch, width, page, heads, dim, q_heads, batch * each, each)
    assert got <= room + 128 * MIB, (got / MIB, room / MIB)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("batch,heads,q_heads", [(1, 8, 32), (1, 1, 32), (40, 8, 8), (3, 2, 2), (5000, 1, 4)])
def test_results_of_single_tokens(batch, heads, q_heads, bits):
    assert need(bits, batch, 500, 16, heads, 128, q_heads, batch, 1) <= 128 * MIB


@pytest.mark.parametrize("bits", [32, 8])
def test_results_of_padding(bits):
    """A hundred thousand tokens that no sequence has, beside two."""
    assert need(bits, 2, 500, 16, 8, 128, 32, 100000, 2) <= 13 * MIB


@pytest.mark.parametrize("bits", [32, 8])
def test_long_prompts_take_what_their_parts_take(bits):
    """Two prompts of 8192 tokens, 32 heads on 8 of 128: no range is cut but for the few rows that single tokens in their
    place would have, 3 workgroups a CU (768, of 256 CUs) of 32 rows: 24576 results of 130 floats."""
    sizes = (2, 600, 16, 8, 128, 32)
    assert need(bits, *sizes, 2 * 8192, 8192) - parts(bits, *sizes, 2 * 8192) <= 13 * MIB
