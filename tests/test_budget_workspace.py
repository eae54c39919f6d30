"""How large the workspaces of a cache under a budget are; no GPU."""

import pytest

from polarquant_kv import _lib


def weights(B, Hq, Hkv, Sq, S, d, qjl):
    return _lib.lib().pqkv_attn_weights_workspace_bytes(B, Hq, Hkv, Sq, S, d, qjl)


@pytest.mark.parametrize("B,Hq,Hkv,Sq,S,d", [(1, 32, 8, 8191, 8191, 128), (8, 32, 8, 8192, 131072, 128),
                                             (1, 64, 8, 32768, 32768, 128), (64, 14, 2, 4096, 4096, 64)])
def test_rotated_queries_have_room_only_with_signs(B, Hq, Hkv, Sq, S, d):
    """Without signs the queries are rotated on their way into the rows'
    records, whose room (two halves of 2 bytes a coordinate, in passes of at most
    512 MB) grows no further with the chunk."""
    rotated = B * Hq * Sq * d * 4
    plain, signed = weights(B, Hq, Hkv, Sq, S, d, 0), weights(B, Hq, Hkv, Sq, S, d, 1)
    assert plain < min(1 << 30, 2 * rotated + (256 << 20))
    assert 2 * rotated < signed < 2 * rotated + (1 << 30)
    assert weights(4 * B, Hq, Hkv, 4 * Sq, S, d, 0) < 1 << 30


@pytest.mark.parametrize("qjl", [0, 1])
@pytest.mark.parametrize("B,Hq,Hkv", [(1, 1, 1), (1, 64, 1), (4, 32, 8), (64, 32, 8), (128, 32, 8), (400, 14, 2)])
def test_bound_past_the_rotated_queries(B, Hq, Hkv, qjl):
    streams = B * Hkv
    for Sq in (1, 32, 257, 8192):
        for S in (1, 127, 8191, 131072, 1048576):
            for d in (64, 128):
                n = weights(B, Hq, Hkv, Sq, S, d, qjl)
                assert n > 0 or streams * -(-S // 128) > 1 << 24
                rotated = 2 * qjl * (B * Hq * Sq * d * 4 + 256)
                assert n <= rotated + (1 << 30) + streams * (4 * S + (128 << 10)), (Sq, S, d, n)


@pytest.mark.parametrize("qjl", [0, 1])
def test_least_workspace(qjl):
    """Smaller where the chunk can run in more passes; what is below it is refused
    (and no address is read for that)."""
    L, fake = _lib.lib(), 0x1000

    def least(*a):
        return L.pqkv_attn_weights_workspace_least_bytes(*a, qjl)

    for a in ((1, 8, 2, 1, 1, 64), (1, 8, 2, 300, 1000, 128), (2, 14, 2, 65, 4096, 64), (8, 32, 8, 8192, 131072, 128),
              (1, 64, 1, 600, 262144, 64)):
        assert 0 < least(*a) <= weights(*a, qjl)
        B, Hq, Hkv, Sq, S, d = a
        for wsb in (0, least(*a) - 1):
            assert L.pqkv_attn_weights(fake, 1, fake, fake, fake, 4, fake if qjl else None, fake if qjl else None,
                                       d if qjl else 0, B, Hq, Hkv, Sq, S - Sq, S, S, d, 0.1, 1, None, 0, fake, S, fake, wsb,
                                       None) == _lib.ERR_WORKSPACE
    rotated = 2 * qjl * 8 * 32 * 8192 * 128 * 4
    assert least(8, 32, 8, 8192, 131072, 128) - rotated < (weights(8, 32, 8, 8192, 131072, 128, qjl) - rotated) / 4
    assert least(1, 8, 3, 4, 16, 128) == 0
