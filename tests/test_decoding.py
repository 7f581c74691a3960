"""CPU: the oracle of the decoding operators against plain torch, and the refusals, in Python and through the C ABI (which
answers before it launches anything)."""
import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import decoding as od


def test_oracle_select_matches_torch_topk():
    g = torch.Generator().manual_seed(1)
    x, s = torch.randn((4, 5, 301), generator=g, dtype=torch.float64), torch.randn((4, 5), generator=g, dtype=torch.float64)
    value = (s.unsqueeze(2) + torch.log_softmax(x, 2)).view(4, -1)
    best = torch.topk(value, 10, dim=1)
    got = od.select(x.numpy(), s.numpy())
    assert np.allclose(got[3], best.values.numpy(), rtol=0, atol=1e-12)
    assert np.array_equal(got[5] * 301 + got[4], best.indices.numpy())
    assert np.array_equal(got[0], got[3][:, :5])  # no end token: the first K


def test_oracle_select_ties_dead_beams_and_end_tokens():
    x = np.zeros((1, 3, 4))
    got = od.select(x, np.array([[-1.0, -1.0, -np.inf]]))
    assert (got[5] * 4 + got[4]).tolist() == [[0, 1, 2, 3, 4, 5]]  # all equal: by index; beam 2 is dead
    got = od.select(x, np.array([[-1.0, -1.0, -np.inf]]), eos=1)
    assert (got[2] * 4 + got[1]).tolist() == [[0, 2, 3]]
    x[0, 0, 2] = np.nan  # the whole beam is out
    got = od.select(x, np.array([[-1.0, -1.0, -1.0]]))
    assert (got[5] * 4 + got[4]).tolist() == [[4, 5, 6, 7, 8, 9]]
    got = od.select(np.full((1, 2, 3), -np.inf), np.zeros((1, 2)))
    assert np.isneginf(got[3]).all() and (got[5] * 3 + got[4]).tolist() == [[0, 1, 2, 3]]


def test_oracle_rounding_is_e4m3():
    """All 256 codes are fixed points, and every float goes where torch's own conversion puts it."""
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy().astype(np.float64)
    assert np.array_equal(od.round_e4m3(codes), codes, equal_nan=True)
    x = torch.randn(20000, generator=torch.Generator().manual_seed(2)) * torch.exp2(torch.randint(-14, 8, (20000,)).float())
    x = x.clamp(-448, 448)
    assert np.array_equal(od.round_e4m3(x.numpy()), x.to(torch.float8_e4m3fn).float().numpy())
    finite = np.sort(np.unique(codes[np.isfinite(codes)]))
    mid = (finite[1:] + finite[:-1]) / 2  # exact ties
    assert np.array_equal(od.round_e4m3(mid), torch.from_numpy(mid).float().to(torch.float8_e4m3fn).double().numpy())


def test_oracle_exponent():
    for most in (448.0, 449.0, 1.75, 1.7500001, 2.0 ** -70, 3e38, 1e-40, 0.0, 7.0, 7.01):
        e = od.exponent(np.array([most, -most / 3, np.nan, -np.inf]))
        assert e == od.EXP_MIN or most <= 448 * 2.0 ** e or e == od.EXP_MAX
        assert e == od.EXP_MIN or most > 448 * 2.0 ** (e - 1)


def test_oracle_cache_shares_copies_and_frees():
    c = od.Cache(4, 200, 1, 2, num_pages=9)
    c.extend([70, 0], every=2)
    assert c.table[0, :2].tolist() == [0, 1] and (c.lens == [70, 0, 0, 0]).all()
    c.write(np.arange(280.0).reshape(2, 70, 1, 2) / 10, np.ones((2, 70, 1, 2)), every=2)
    c.reorder([[0, 0], [-1, -1]])
    assert c.refs[:3].tolist() == [2, 2, 0]
    c.extend([1, 1, 0, 0])  # both beams write into page 1: the first keeps it
    assert c.table[:2, :2].tolist() == [[0, 1], [0, 2]] and c.refs[:3].tolist() == [2, 1, 1]
    assert np.array_equal(c.tokens(0, 0, 0, 0)[:70], c.tokens(1, 0, 0, 0)[:70])
    c.reorder([[1, 1], [0, 1]])
    assert c.refs[:3].tolist() == [2, 0, 2]
    assert c.compact() == 2 and c.table[:2, :2].tolist() == [[0, 1], [0, 1]]
    c.extend(1000)
    assert c.status == 2 and (c.lens == c.starts).all()


def test_oracle_attention_is_softmax():
    rng = np.random.default_rng(3)
    c = od.Cache(1, 100, 1, 64)
    c.extend(80)
    k, v, q = (rng.standard_normal((1, 80, 1, 64)) for _ in range(3))
    c.write(k, v)
    kk, vv = (torch.from_numpy(c.tokens(0, 0, 0, w)) for w in range(2))
    want = torch.nn.functional.scaled_dot_product_attention(torch.from_numpy(q[:, :, 0])[None], kk[None, None], vv[None, None], is_causal=True)
    assert np.allclose(c.attend(q)[0, :, 0], want[0, 0].numpy(), atol=1e-12)
    assert np.abs(kk.numpy() - k[0, :, 0]).max() <= 2.0 ** -4 * np.abs(k).max()


# ---- refusals


def test_refusals_without_a_gpu():
    from asr_amd import _lib
    from asr_amd.decoding import PagedKVCache, beam_select, reorder_states

    logits, scores = torch.zeros((10, 7)), torch.zeros((2, 5))
    with pytest.raises(_lib.AsrkError):
        beam_select(logits, scores)
    with pytest.raises(ValueError):
        beam_select(logits, scores.double())
    with pytest.raises(ValueError):
        beam_select(logits[:9], scores)
    with pytest.raises(ValueError):
        beam_select(logits.half(), scores)
    with pytest.raises(ValueError):
        beam_select(torch.zeros((2, 5, 1)), scores)
    with pytest.raises(ValueError):
        beam_select(torch.zeros((17, 7)), torch.zeros((1, 17)))
    with pytest.raises(ValueError):
        reorder_states(torch.zeros((2, 5, 3)), torch.zeros((2, 5), dtype=torch.int32))
    with pytest.raises(ValueError):
        reorder_states(torch.zeros((3, 5, 3)), torch.zeros((2, 5), dtype=torch.int64))
    with pytest.raises(_lib.AsrkError):
        reorder_states(torch.zeros((2, 5, 3)), torch.zeros((2, 5), dtype=torch.int64))
    with pytest.raises(_lib.AsrkError):
        PagedKVCache(2, 100, 1, 64, device="cpu")
    for bad in (dict(num_seqs=0), dict(max_len=0), dict(kv_heads=0), dict(head_dim=96), dict(num_layers=0), dict(num_pages=0)):
        with pytest.raises(ValueError):
            PagedKVCache(**{**dict(num_seqs=2, max_len=100, kv_heads=1, head_dim=64), **bad})


def _cache_struct(**over):
    from asr_amd import _lib

    at = 1 << 20  # never dereferenced
    f = dict(num_layers=2, num_pages=8, kv_heads=2, head_dim=64, num_seqs=4, max_pages=2, seq_stride=1,
             **{n: at for n in ("kv", "exps", "table", "lens", "starts", "refs", "status", "scratch")})
    f.update(over)
    return ctypes.byref(_lib.KVCache(**{k: (ctypes.c_void_p(v) if k not in dict(_lib.KVCache._fields_[:7]) else v) for k, v in f.items()}))


NULL, SHAPE, ALIGN, WORKSPACE, UNSUPPORTED = -1, -2, -3, -5, -6


def test_c_abi_refusals():
    from asr_amd import _lib

    lib = _lib.load()
    p = 1 << 20
    c = _cache_struct()
    for name in ("kv", "exps", "table", "lens", "starts", "refs", "status", "scratch"):
        assert lib.asrk_kv_extend(_cache_struct(**{name: 0}), None, 1, None) == NULL, name
    for over in (dict(num_layers=0), dict(num_pages=0), dict(kv_heads=0), dict(head_dim=80), dict(num_seqs=0), dict(max_pages=0),
                 dict(seq_stride=0), dict(num_seqs=70000), dict(max_pages=1 << 30)):
        assert lib.asrk_kv_extend(_cache_struct(**over), None, 1, None) == SHAPE, over
        assert lib.asrk_kv_attention_workspace_bytes(_cache_struct(**over), 1, 2, 1) == 0
    assert lib.asrk_kv_extend(None, None, 1, None) == NULL
    assert lib.asrk_kv_extend(_cache_struct(kv=p + 8), None, 1, None) == ALIGN
    assert lib.asrk_kv_extend(c, None, -1, None) == SHAPE
    assert lib.asrk_kv_reorder(c, None, 2, None) == NULL
    assert lib.asrk_kv_reorder(c, p, 3, None) == SHAPE and lib.asrk_kv_reorder(c, p, 0, None) == SHAPE
    assert lib.asrk_kv_reorder(_cache_struct(num_seqs=33), p, 33, None) == SHAPE
    assert lib.asrk_kv_compact(_cache_struct(seq_stride=2), None) == SHAPE

    def write(layer=0, k=p, v=p, dt=_lib.ASRK_BF16, lds=(128, 128, 64), n=1):
        return lib.asrk_kv_write(c, layer, k, v, dt, *lds, n, None)

    assert write(k=None) == NULL and write(v=None) == NULL and write(dt=_lib.ASRK_I16) == UNSUPPORTED
    assert write(layer=2) == SHAPE and write(layer=-1) == SHAPE and write(n=0) == SHAPE and write(lds=(-8, 8, 8)) == SHAPE
    assert write(k=p + 2) == ALIGN and write(lds=(128, 4, 64)) == ALIGN

    def read(layer=0, layers=2, count=5, k=p, v=p):
        return lib.asrk_kv_read(c, layer, layers, None, 0, count, k, v, None)

    assert read(k=None) == NULL and read(layers=3) == SHAPE and read(layer=1) == SHAPE and read(count=0) == SHAPE and read(v=p + 4) == ALIGN

    def attend(layer=0, q=p, lds=(256, 128, 64), n=1, heads=4, beams=1, out=p, ws=p, ws_bytes=1 << 30):
        return lib.asrk_kv_attention(c, layer, q, *lds, n, heads, beams, 0.125, out, ws, ws_bytes, None)

    assert attend(q=None) == NULL and attend(out=None) == NULL and attend(layer=2) == SHAPE and attend(n=0) == SHAPE
    assert lib.asrk_kv_attention(c, 0, p, 256, 128, 64, 1, 4, 1, 0.0, p, p, 1 << 30, None) == SHAPE
    assert lib.asrk_kv_attention(c, 0, p, 256, 128, 64, 1, 4, 1, float("nan"), p, p, 1 << 30, None) == SHAPE
    assert attend(heads=3) == SHAPE and attend(heads=0) == SHAPE and attend(beams=3) == SHAPE and attend(beams=0) == SHAPE
    assert attend(lds=(256, 4, 64)) == ALIGN and attend(out=p + 8) == ALIGN
    big = _cache_struct(max_pages=100)
    need = lib.asrk_kv_attention_workspace_bytes(big, 1, 4, 1)
    assert need > 0
    assert lib.asrk_kv_attention(big, 0, p, 256, 128, 64, 1, 4, 1, 0.125, p, None, 0, None) == NULL
    assert lib.asrk_kv_attention(big, 0, p, 256, 128, 64, 1, 4, 1, 0.125, p, p, need - 1, None) == WORKSPACE

    def select(logits=p, dt=_lib.ASRK_F32, ld=100, B=2, K=5, V=100, ws=p, ws_bytes=1 << 30, out=p):
        return lib.asrk_beam_select(logits, dt, ld, p, B, K, V, -1, out, p, p, p, p, p, ws, ws_bytes, None)

    assert select(logits=None) == NULL and select(out=None) == NULL and select(ws=None) == NULL and select(dt=_lib.ASRK_I16) == UNSUPPORTED
    for over in (dict(B=0), dict(K=0), dict(K=17), dict(V=1), dict(ld=99), dict(B=20000), dict(K=16, V=1 << 21, ld=1 << 21)):
        assert select(**over) == SHAPE, over
    assert select(logits=p + 1) == ALIGN and select(ws=p + 8) == ALIGN and select(ws_bytes=16) == WORKSPACE
    assert lib.asrk_beam_select_workspace_bytes(2, 17, 100) == 0
    assert lib.asrk_reorder_rows(None, p, 2, 5, 16, p, None) == NULL
    assert lib.asrk_reorder_rows(p, p, 2, 5, 0, p, None) == SHAPE and lib.asrk_reorder_rows(p, p, 20000, 5, 16, p, None) == SHAPE
    assert math.isfinite(need)


def test_c_abi_refuses_more_columns_than_the_grid_takes():
    from asr_amd import _lib

    lib = _lib.load()
    p, c = 1 << 20, _cache_struct(max_pages=100)
    most = 65535 * 128 // 2  # of two query heads per key/value head
    for n, beams, want in ((most, 1, NULL), (most + 1, 1, SHAPE), (most // 2, 2, NULL), (most // 2 + 1, 2, SHAPE)):  # NULL: the shape is taken
        assert lib.asrk_kv_attention(c, 0, None, 256, 128, 64, n, 4, beams, 0.125, p, p, 1 << 60, None) == want, (n, beams)
