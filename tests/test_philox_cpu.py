"""The counter-based generator against the answers published with it (Random123's kat_vectors, Philox-4x32 with ten rounds)."""
import pytest
import torch

from system_lab_b200.ops import reference as ref

ONES, PI = (0xFFFFFFFF,) * 6, (0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344, 0xA4093822, 0x299F31D0)


@pytest.mark.parametrize("given,want", [((0,) * 6, (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
                                        (ONES, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
                                        (PI, (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))], ids=["zeros", "ones", "pi"])
def test_published_answers(given, want):
    """Four words of counter and two of key, low ones first: each has its place."""
    c0, c1, c2, c3, k0, k1 = given
    block = c0 | c1 << 32
    words = ref.philox_words(torch.tensor([block - (1 << 64) if block >> 63 else block]), k0 | k1 << 32, c2 | c3 << 32)
    assert tuple(int(w) for w in words) == want


def test_bits_are_halves_of_words():
    a, b = ref.philox_bits(24, 7, 2 ** 40 + 3), ref.philox_words(torch.arange(3), 7, 2 ** 40 + 3)
    for e in range(24):
        word = int(b[e % 8 // 2][e // 8])
        assert int(a[e]) == (word >> 16 if e % 2 else word & 0xFFFF)
