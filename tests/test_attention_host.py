"""Kernel attention: what it refuses, before anything reaches a device."""
import ctypes

import pytest
import torch

import rapidalign_b200 as ra
from rapidalign_b200 import _lib


def qkv(n=5, m=7, h=4, hk=2, d=8, dtype=torch.float32):
    return (torch.zeros(n, h, d, dtype=dtype), torch.zeros(m, hk, d, dtype=dtype),
            torch.zeros(m, hk, d, dtype=dtype))


@pytest.mark.parametrize("change, message", [
    (lambda q, k, v: ((q[0], k, v), {}), "must have shape"),
    (lambda q, k, v: ((q, k[:3], v), {}), "same shape"),
    (lambda q, k, v: ((q[..., :4], k, v), {}), "same head dimension"),
    (lambda q, k, v: ((q.half(), k, v), {}), "share dtype"),
    (lambda q, k, v: ((q.double(), k.double(), v.double()), {}), "share dtype"),
    (lambda q, k, v: ((q[:, :3], k, v), {}), "multiple"),
    (lambda q, k, v: ((q[..., :0], k[..., :0], v[..., :0]), {}), "between 1 and 256"),
    (lambda q, k, v: ((q, k, v), {"scale": float("nan")}), "scale"),
    (lambda q, k, v: ((q, k, v), {"softcap": -2.0}), "softcap"),
    (lambda q, k, v: ((q, k, v), {"softcap": 1e-7}), "softcap"),
    (lambda q, k, v: ((q, k, v), {"softcap": float("inf")}), "softcap"),
])
def test_refuses(change, message):
    args, kw = change(*qkv())
    with pytest.raises(ValueError, match=message):
        ra.pyg_kernel_attention(*args, q_ptr=torch.tensor([0, 5]), k_ptr=torch.tensor([0, 7]), **kw)
    with pytest.raises(ValueError, match=message):
        ra.kernel_attention_dense(*(t[None] for t in args), **kw)


def test_wide_heads_are_refused():
    with pytest.raises(ValueError, match="between 1 and 256"):
        ra.kernel_attention_dense(*(t[None] for t in qkv(d=257)))


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        ra.pyg_kernel_attention(*qkv(), q_ptr=torch.tensor([0, 5]), k_ptr=torch.tensor([0, 7]))
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        ra.kernel_attention_dense(*(t[None] for t in qkv()))
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        ra.attention_segments(torch.tensor([0, 5]))
    with pytest.raises(ValueError, match="either ptr or batch"):
        ra.attention_segments()


@pytest.mark.parametrize("kw, message", [
    (dict(k_pos=torch.zeros(7, 3)), "go together"),
    (dict(sigma=1.0), "go together"),
    (dict(q_pos=torch.zeros(5, 3), k_pos=torch.zeros(7, 3)), "need a sigma"),
    (dict(q_pos=torch.zeros(5, 3), k_pos=torch.zeros(7, 3), sigma=0.0), "must be positive"),
    (dict(q_pos=torch.zeros(5, 3), k_pos=torch.zeros(7, 3), sigma=float("nan")), "positive"),
    (dict(q_pos=torch.zeros(5, 4), k_pos=torch.zeros(7, 4), sigma=1.0), "1 to 3"),
    (dict(q_pos=torch.zeros(5, 3), k_pos=torch.zeros(7, 2), sigma=1.0), "1 to 3"),
    (dict(q_pos=torch.zeros(5, 3), sigma=1.0), "length"),
    (dict(q_pos=torch.zeros(1, 5, 3), k_pos=torch.zeros(1, 7, 3), sigma=1.0), "1 to 3"),
    (dict(q_pos=torch.zeros(5, 3).long(), k_pos=torch.zeros(7, 3).long(), sigma=1.0), "floating"),
    (dict(q_pos=torch.zeros(5, 3), k_pos=torch.zeros(7, 3), sigma=torch.ones(3)), "per head"),
])
def test_positions_are_checked(kw, message):
    from rapidalign_b200.attention import _positions
    args = [kw.get(n) for n in ("q_pos", "k_pos", "sigma")]
    with pytest.raises(ValueError, match=message):
        _positions(*args, (5,), (7,), 4, torch.device("cpu"))


def test_tiles():
    """Every 128 rows of every graph once, the costly graphs first."""
    from rapidalign_b200.attention import _tiles
    lengths = torch.tensor([0, 1, 128, 129, 300])
    other = torch.tensor([9, 5, 7, 5, 100])
    first, ofirst = lengths.cumsum(0) - lengths, other.cumsum(0) - other
    got = _tiles(first, lengths, ofirst, other, 7)
    assert got.dtype == torch.int32
    assert got.tolist() == [[258, 128, 26, 100], [386, 128, 26, 100], [514, 44, 26, 100],
                            [1, 128, 14, 7], [0, 1, 9, 5], [129, 128, 21, 5], [257, 1, 21, 5]]
    empty = _tiles(torch.tensor([0, 0]), torch.tensor([0, 0]), first[:2], other[:2], 0)
    assert empty.shape == (0, 4)


@pytest.fixture(scope="module")
def lib():
    from rapidalign_b200 import build as b
    b.build()
    return _lib.load()


def desc(**kw):
    word = ctypes.c_int32(0)
    d = _lib.RaAttnDesc(graphs=2, num_q=100, num_k=100, max_q=60, max_k=60, q_tiles=2, k_tiles=2,
                        q_row=256, q_head=64, k_row=256, k_head=64, v_row=256, v_head=64, heads=4,
                        kv_heads=4, dim=64, pos_dim=3, dtype=_lib.RA_BF16, scale=0.125,
                        softcap=0.0, status=ctypes.addressof(word))
    d.keep = word
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def test_c_sizes(lib):
    assert lib.ra_attn_workspace_bytes(ctypes.byref(desc()), 0) >= 256
    assert lib.ra_attn_workspace_bytes(ctypes.byref(desc()), 1) >= 36 * 400
    assert lib.ra_attn_workspace_bytes(ctypes.byref(desc(num_q=0, num_k=0, max_q=0, max_k=0,
                                                         q_tiles=0, k_tiles=0, graphs=0)), 1) >= 256


@pytest.mark.parametrize("bad", [
    dict(graphs=-1), dict(num_q=-1), dict(num_k=2 ** 31), dict(heads=3, kv_heads=2),
    dict(heads=0), dict(kv_heads=0), dict(dim=0), dict(dim=257), dict(pos_dim=4),
    dict(dtype=3), dict(softcap=-1.0), dict(scale=float("inf")), dict(q_row=-1),
    dict(max_q=101), dict(status=None), dict(num_q=2 ** 30, heads=8),
])
def test_c_refuses(lib, bad):
    d = desc(**bad)
    assert lib.ra_attn_workspace_bytes(ctypes.byref(d), 0) == 0
    base = 1 << 20
    inp = _lib.RaAttnInputs(*[base] * 12)
    rc = lib.ra_attn_forward(ctypes.byref(d), ctypes.byref(inp), base, base, base, base, 1 << 30,
                             base, 1 << 30, None)
    assert rc == _lib.RA_ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("missing", ["q", "k", "v", "q_pos", "k_pos", "sigma", "k_ptr", "q_tiles"])
def test_c_refuses_missing_inputs(lib, missing):
    base = 1 << 20  # never touched: the checks come first
    d = desc()
    inp = _lib.RaAttnInputs(*[base] * 12)
    setattr(inp, missing, None)
    rc = lib.ra_attn_forward(ctypes.byref(d), ctypes.byref(inp), base, base, base, base, 1 << 30,
                             base, 1 << 30, None)
    assert rc == _lib.RA_ERR_INVALID_ARGUMENT


def test_c_refuses_buffers(lib):
    base = 1 << 20
    d = desc()
    inp = _lib.RaAttnInputs(*[base] * 12)
    big = 1 << 30
    for state, n_state, ws, n_ws in ((base + 8, big, base, big), (base, 16, base, big),
                                     (base, big, base + 8, big), (base, big, base, 16)):
        assert lib.ra_attn_forward(ctypes.byref(d), ctypes.byref(inp), base, base, base, state,
                                   n_state, ws, n_ws, None) == _lib.RA_ERR_WORKSPACE
    assert lib.ra_attn_forward(ctypes.byref(d), ctypes.byref(inp), base + 2, base, base, base,
                               big, base, big, None) == _lib.RA_ERR_INVALID_ARGUMENT
    gr = _lib.RaAttnGrads(*[base] * 6)
    assert lib.ra_attn_backward(ctypes.byref(d), ctypes.byref(inp), base, None, base, base,
                                ctypes.byref(gr), base, big, base, 256,
                                None) == _lib.RA_ERR_WORKSPACE
    d.pos_dim = 0
    assert lib.ra_attn_backward(ctypes.byref(d), ctypes.byref(inp), base, None, base, base,
                                ctypes.byref(gr), base, big, base, big,
                                None) == _lib.RA_ERR_INVALID_ARGUMENT
    # padded clouds: the counts have to fit
    inp = _lib.RaAttnInputs(*[base] * 12)
    inp.q_ptr = inp.k_ptr = None
    assert lib.ra_attn_forward(ctypes.byref(desc()), ctypes.byref(inp), base, base, base, base,
                               big, base, big, None) == _lib.RA_ERR_INVALID_ARGUMENT
