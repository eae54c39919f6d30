"""Arguments that the kernels would read past, refused before any launch; no GPU."""

import pytest
import torch

from polarquant_kv import attention
from polarquant_kv.types import PagedPQCache, PQCache

D = 64


def caches(paged, jl_dim=D):
    out = []
    for signs in (jl_dim, 0):
        if paged:
            c = PagedPQCache(1, 2, D, 4, torch.zeros(16), "cpu", 64, jl_dim=signs)
            c.ensure(8)
            c.seq_len = 8
        else:
            c = PQCache(blocks=torch.zeros(1, 2, 8, 36, dtype=torch.uint8), head_dim=D, n_bits=4, seq_len=8, max_seq_len=8,
                        codebooks=torch.zeros(16), jl_dim=signs,
                        qjl_signs=torch.zeros(1, 2, 8, max(signs, 64) // 8, dtype=torch.uint8) if signs else None)
        out.append(c)
    return out


def calls(kc, vc, jl_rot):
    q, R = torch.zeros(1, 4, D), torch.eye(D)
    yield lambda: attention.decode_attention_weights(q, kc, vc, R, jl_rot=jl_rot)
    yield lambda: attention.attention_weights(q.unsqueeze(2), kc, R, 7, jl_rot=jl_rot)
    yield lambda: attention.decode_attention(q, kc, vc, R, jl_rot=jl_rot)
    yield lambda: attention.prefill_attention(q.unsqueeze(2), kc, vc, R, 7, jl_rot=jl_rot)


@pytest.mark.parametrize("paged", [False, True])
def test_projections_of_another_size(paged):
    kc, vc = caches(paged)
    for shape in ((32, D), (D, 32), (128, D), (D,)):
        for call in calls(kc, vc, torch.zeros(shape)):
            with pytest.raises(ValueError, match="jl_rot must be"):
                call()
    for call in calls(kc, vc, torch.zeros(D, D)):               # as they should be: on to the next check
        with pytest.raises(ValueError, match="device tensors"):
            call()
    for call in calls(vc, vc, torch.zeros(D, D)):
        with pytest.raises(ValueError, match="no signs"):
            call()
    kc, vc = caches(paged, 128)
    for call in calls(kc, vc, torch.zeros(D, D)):
        with pytest.raises(ValueError, match="projections"):
            call()


def adopted(width, pages):
    c = PagedPQCache(1, 2, D, 4, torch.zeros(16), "cpu", 64, jl_dim=D)
    table, signs = (torch.arange(2 * width).view(2, width) + o for o in (1000, 2000))
    c.adopt(table, pages * 64, [], signs)
    c.seq_len = 40
    return c, table, signs


@pytest.mark.parametrize("widths", [(2, 5), (5, 2)])
def test_tables_of_the_caller_stay_the_callers(widths):
    """What their owner writes into them later is what later calls read."""
    (keys, kt, ks), (values, vt, _) = (adopted(w, 1) for w in widths)
    attention.check_paged(1, 4, D, keys, values)
    assert keys.table is kt and values.table is vt and keys.sign_table is ks
    for _ in range(2):
        k, v, s, n = attention.page_tables(keys, values)
        assert n == 5 and all(t.shape == (2, 5) and t.is_contiguous() for t in (k, v, s))
        assert torch.equal(k[:, :kt.shape[1]], kt) and torch.equal(v[:, :vt.shape[1]], vt)
        assert torch.equal(s[:, :ks.shape[1]], ks)
        kt[1, 1], vt[1, 1], ks[1, 1] = 77, 78, 79               # the owner's next page


def test_caches_that_are_views():
    """Rows that do not follow each other would be read as if they did."""
    kc, vc = caches(False)
    wide = torch.zeros(1, 2, 20, 36, dtype=torch.uint8)
    view = PQCache(blocks=wide[:, :, :8], head_dim=D, n_bits=4, seq_len=8, max_seq_len=8, codebooks=torch.zeros(16))
    signs = PQCache(blocks=kc.blocks, head_dim=D, n_bits=4, seq_len=8, max_seq_len=8, codebooks=torch.zeros(16), jl_dim=D,
                    qjl_signs=torch.zeros(1, 2, 20, 8, dtype=torch.uint8)[:, :, :8])
    for bad, jl_rot in ((view, None), (signs, torch.zeros(D, D))):
        for call in calls(bad, vc, jl_rot):
            with pytest.raises(ValueError, match="contiguous"):
                call()
    for call in calls(signs, vc, None):                          # nothing reads them: on to the next check
        with pytest.raises(ValueError, match="device tensors"):
            call()
