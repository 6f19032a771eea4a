"""What the softmax operators ask of memory (C entries; no device)."""
import ctypes

import pytest

from rapidalign_b200 import _lib
from test_attention_host import desc as attn_desc
from test_cross_entropy_host import desc as ce_desc


@pytest.fixture(scope="module")
def lib():
    from rapidalign_b200 import build as b
    b.build()
    return _lib.load()


@pytest.mark.parametrize("dtype", [_lib.RA_F32, _lib.RA_BF16, _lib.RA_F16])
@pytest.mark.parametrize("rows", [9, 8192, 32768, 1 << 20])
@pytest.mark.parametrize("vocab", [1000, 131072, 1 << 20, 1 << 24])
def test_no_logits_in_the_forward(lib, rows, vocab, dtype):
    """The partials of a pass stay below 128 MiB (one tile of rows where the table
    alone is longer than that allows); 12 bytes a row besides."""
    d = ce_desc(rows=rows, vocab=vocab, dtype=dtype)
    part = max(128 << 20, 128 * 8 * 4 * -(-vocab // 128))
    assert lib.ra_ce_workspace_bytes(ctypes.byref(d), 0) <= part + 12 * rows + (1 << 20)


@pytest.mark.parametrize("rows", [1, 5, 8])
def test_few_rows_keep_no_copy_of_the_table(lib, rows):
    d = ce_desc(rows=rows, vocab=131072, dim=1024, ld_x=1024, ld_w=1024, dtype=_lib.RA_F32)
    assert lib.ra_ce_state_bytes(ctypes.byref(d)) > 4 * 131072 * 1024
    d.forward_only = 1
    assert lib.ra_ce_state_bytes(ctypes.byref(d)) < 4096
    d.rows = 9  # the product kernel reads the halves
    assert lib.ra_ce_state_bytes(ctypes.byref(d)) > 4 * 131072 * 1024


def test_few_queries_keep_no_copy_of_the_keys(lib):
    kw = dict(graphs=1, num_q=1, max_q=1, q_tiles=1, num_k=100000, max_k=100000, k_tiles=782,
              dtype=_lib.RA_F32)
    d = attn_desc(**kw)
    assert lib.ra_attn_state_bytes(ctypes.byref(d)) > 2 * 4 * 100000 * 256
    d.forward_only = 1
    assert lib.ra_attn_state_bytes(ctypes.byref(d)) <= 256
    d.num_q = d.max_q = 9
    assert lib.ra_attn_state_bytes(ctypes.byref(d)) > 2 * 4 * 100000 * 256


def test_forward_only_is_checked(lib):
    base, big = 1 << 20, 1 << 40
    d = attn_desc(dtype=_lib.RA_F32, graphs=1, num_q=1, max_q=1, q_tiles=1, forward_only=1)
    inp = _lib.RaAttnInputs(*[base] * 12)
    gr = _lib.RaAttnGrads(*[base] * 6)

    def forward(stats=None):
        return lib.ra_attn_forward(ctypes.byref(d), ctypes.byref(inp), base, base, stats, base,
                                   big, base, big, None)

    assert forward(stats=base) == _lib.RA_ERR_INVALID_ARGUMENT
    inp.k = base + 4  # operands off the boundary would need halves
    assert forward() == _lib.RA_ERR_INVALID_ARGUMENT
    inp.k, d.k_row = base, 258
    assert forward() == _lib.RA_ERR_INVALID_ARGUMENT
    assert lib.ra_attn_backward(ctypes.byref(d), ctypes.byref(inp), base, base, None, base,
                                ctypes.byref(gr), base, big, base, big, None) == _lib.RA_ERR_STATE
    d.forward_only = 2
    assert lib.ra_attn_state_bytes(ctypes.byref(d)) == 0

    c = ce_desc(rows=3, dtype=_lib.RA_F32, forward_only=1)
    assert lib.ra_ce_backward(ctypes.byref(c), base, base, base, base, None, base, base, base, big,
                              base, big, None) == _lib.RA_ERR_STATE
    c.forward_only = 2
    assert lib.ra_ce_state_bytes(ctypes.byref(c)) == 0
