"""What the token stage's entry points refuse by size, without a GPU: a call that is not refused would fail at its launch,
with an error above 0."""
import ctypes

import pytest

from pigeon_amd import _lib


@pytest.fixture
def p():
    buf = ctypes.create_string_buffer(64)
    yield (ctypes.addressof(buf) + 15) & ~15


def test_launches_of_two_to_the_32_threads_are_refused(p):
    lib = _lib.load()
    sample = lambda B: lib.pgn_sample_tokens(p, 0, 6, B, 6, p, None, 1.0, None, 0, None, 1.0, None, 0.0, p, None)              # noqa: E731
    assert sample(1 << 22) == -2 and sample((1 << 31) - 1) == -2

    def attend(T, R, Hkv, starts):                                  # a table of one page: nothing is split, no workspace
        return lib.pgn_cached_attention(p, 1, p, p, p, p, p, 1, p, starts, p, T, R, Hkv, Hkv, 64, 4, 1, 16, 64 * Hkv, 64, 64 * Hkv, 64, 0.1, 1, 0,
                                        None, 0, None)
    for R, Hkv in ((1 << 24, 1), (1 << 19, 32), ((1 << 18) + 1, 64)):
        assert attend(R, R, Hkv, None) == -2                        # single tokens, a tile each
    assert attend(1 << 24, 1 << 22, 1, p) == -2                     # packed: four tiles of 16 rows a request
    assert attend(1 << 26, 1, 32, p) == -2                          # one prompt: 2^19 tiles of 128 rows and one, of 32 heads

    def write(T, H):
        return lib.pgn_cache_write(p, p, 1, p, T, H, 64, 64 * H, 64, 64 * H, 64, p, p, p, p, 4, 16, None)
    assert write(1 << 24, 64) == -2 and write(1 << 30, 1) == -2     # 64 tokens a workgroup, for each head
