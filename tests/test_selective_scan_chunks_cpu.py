"""The chunks that the selective scan cuts the sizes of test_selective_scan_chunks_gpu.py into, by the
forward's workspace: for each chunk of a batch entry and channel N states and one sum of d, rows of
B and C besides.  CPU only."""
import pytest

from gdn2_package import _lib

# tokens of a chunk: (B, T, C, G).  For each of four widths of the states; a chunk of 32 or more
# holds several blocks of 16 tokens, T is a multiple of neither
CHUNKED = {16: (3, 137, 40, 4), 32: (8, 300, 48, 16), 64: (32, 300, 64, 32), 128: (64, 300, 96, 32)}
STATES = {5: 8, 16: 16, 24: 32, 64: 64}   # and what they are padded to

# one group of two whole waves' channels and a few more
WIDE = {64: (300, 300, 130, 1), 128: (500, 300, 130, 1)}


@pytest.mark.parametrize("L,size,N", [(L, s, N) for L, s in CHUNKED.items() for N in STATES] +
                         [(L, s, 16) for L, s in WIDE.items()])
def test_chunks(L, size, N):
    B, T, C, G = size
    NP, chunks = STATES[N], -(-T // L)
    assert T % 16 and T % L and chunks > 1
    up = lambda n: (n + 15) // 16 * 16
    want = up(B * chunks * C * NP * 4) + up(B * chunks * C * 4) + up(B * T * G * 2 * NP * 4)
    assert _lib.lib().gdn2_selective_scan_workspace_bytes(B, T, C, G, N, 0) == want
