"""The decoding operators on the GPU against their 64-bit restatement (oracle/decoding.py).

Tolerances.  What is held in the cache, and every whole number, is compared exactly.  Scores: a float32 sum of 32 exponentials
per lane (32 * 2**-24), exponentials of a float32 argument (17 * 1.44 * 2**-24 for the terms that count) and a result of
magnitude below 64 rounded to float32 (2**-19): together below 1e-5.  Attention: half a step of the bfloat16 result (2**-8 of
it), the weights' rounding to 11 bits (2**-11 of sum p |v| / sum p), and float32 sums of products of up to 128 terms in the
scores, a relative 128 * 2**-24 * sum |q k| * scale in the weights, below 2**-12 for the inputs here: 2**-10 for the two.
"""
import math

import numpy as np
import pytest
import torch

from oracle import decoding as od

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def PagedKVCache_(*args, **kw):
    from asr_amd.decoding import PagedKVCache

    return PagedKVCache(*args, **kw)


# ---- selection


def check_select(logits, scores, eos=None):
    from asr_amd.decoding import beam_select

    B, K = scores.shape
    step = beam_select(logits, scores, eos)
    want = od.select(logits.reshape(B, K, -1).double().cpu().numpy(), scores.double().cpu().numpy(), -1 if eos is None else eos)
    got = [t.cpu().numpy() for t in step]
    for i in (1, 2, 4, 5):
        assert got[i].dtype == np.int64 and np.array_equal(got[i], want[i]), (i, got[i], want[i])
    for i in (0, 3):
        assert got[i].dtype == np.float32 and np.allclose(got[i], want[i], rtol=0, atol=1e-5), np.abs(got[i] - want[i]).max()
    return step


@pytest.mark.parametrize("B,K,V,dtype,pad", [
    (1, 1, 2, "f32", 0), (2, 1, 3, "bf16", 0), (3, 2, 2, "f32", 1), (2, 16, 130, "f32", 0), (4, 8, 8192, "bf16", 0), (2, 3, 8193, "f32", 3),
    (1, 5, 49157, "bf16", 59), (3, 5, 51865, "bf16", 0), (1, 16, 20001, "bf16", 0), (2, 7, 70001, "f32", 0), (130, 4, 97, "bf16", 0), (171, 12, 8197, "bf16", 0)])
def test_select(B, K, V, dtype, pad):
    g = _gen(B * 1000 + V)
    x = (torch.randn((B * K, V + pad), generator=g, device="cuda") * 3).to(torch.bfloat16 if dtype == "bf16" else torch.float32)[:, :V]
    s = -torch.rand((B, K), generator=g, device="cuda") * 20
    check_select(x, s)
    check_select(x, s, eos=int(x[0].argmax()))
    if K > 1:
        s[:, 1:] = -math.inf  # the first step
        check_select(x, s, eos=V - 1)
    if pad == 0:
        check_select(x.view(B, K, V), s, eos=0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [2, 2050])
def test_select_rows_that_end_anywhere(rows, dtype):
    """Rows that end within a piece, a wave's share or a chunk, with NaN behind them."""
    g = _gen(rows)
    sizes = [*range(2, 19), 255, 256, 257, 511, 513, 2047, 2051, 4100, 8190, 8191, 8195, 8199, 8200, 16383, 16385, 16391]
    for V in sizes if rows == 2 else (3, 9, 513, 8191, 8199, 8200):
        x = (torch.randn((rows, V + 9), generator=g, device="cuda") * 3).to(torch.bfloat16 if dtype == "bf16" else torch.float32)
        x[:, V:] = math.nan
        s = -torch.rand((rows // 2, 2), generator=g, device="cuda")
        check_select(x[:, :V], s)
        check_select(x.view(-1)[1:1 + rows // 2 * 2 * (V + 8)].view(rows, V + 8)[:, :V].nan_to_num(0.25).contiguous(), s, eos=1)


def test_select_last_position_of_a_run():
    x = torch.randn((6, 4, 1001), generator=_gen(5), device="cuda")
    check_select(x[:, -1], -torch.rand((2, 3), generator=_gen(6), device="cuda"))
    check_select(x.view(2, 3, 4, 1001)[:, :, 2], -torch.rand((2, 3), generator=_gen(7), device="cuda"))


@pytest.mark.parametrize("V", [40, 1024, 16385, 51865])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_select_ties_go_to_the_lowest_index(V, dtype):
    K = 5
    x = torch.zeros((2 * K, V), device="cuda", dtype=dtype)  # equal beams, equal words; odd rows start at odd addresses
    check_select(x, torch.full((2, K), -3.0, device="cuda"))
    x[:, 1::2] = -0.0  # equal to 0
    check_select(x, torch.full((2, K), -3.0, device="cuda"), eos=0)
    row = torch.randn((V,), generator=_gen(V), device="cuda").to(dtype)
    row[V // 2:] = row[:V - V // 2].clone()  # every word twice
    check_select(row.expand(2 * K, V).contiguous(), torch.full((2, K), -3.0, device="cuda"))
    up = torch.arange(V, device="cuda").float().div(V).to(dtype)  # ascending: bf16 has long runs of equal values
    check_select(torch.stack([up, up.flip(0)] * K), torch.linspace(-1, -7, 2 * K, device="cuda").view(2, K))


def test_select_dead_beams():
    g = _gen(11)
    x = torch.randn((4, 4, 9001), generator=g, device="cuda")
    s = -torch.rand((4, 4), generator=g, device="cuda")
    x[0, 1, 17] = math.nan
    x[0, 2, 8999] = math.inf
    x[0, 3] = -math.inf
    s[1, 0], s[1, 1], s[1, 2] = math.nan, math.inf, -math.inf
    x[1, 2] = math.nan  # behind a dead score
    s[2] = -math.inf  # nothing lives
    x[3, :, 5:] = -math.inf  # fewer words than candidates
    x[3, 0, :] = -math.inf
    x[3, 0, 3] = 2.0
    check_select(x.view(16, -1), s)
    check_select(x.view(16, -1), s, eos=3)
    check_select(x.view(16, -1).bfloat16(), s, eos=1)


def test_reorder_states():
    from asr_amd.decoding import reorder_states

    g = _gen(3)
    par = torch.randint(0, 5, (7, 5), generator=g, device="cuda")
    for shape, dtype in (((7, 5, 3, 11), torch.int64), ((35, 13), torch.uint8), ((35,), torch.float32), ((7, 5, 4096), torch.bfloat16), ((35, 100000), torch.int16)):
        x = torch.randint(0, 100, shape, generator=g, device="cuda").to(dtype)
        want = x.reshape(7, 5, -1)[torch.arange(7, device="cuda")[:, None], par].reshape(shape)
        assert torch.equal(reorder_states(x, par), want), (shape, dtype)
    x = torch.randn((7, 5, 6), generator=g, device="cuda")
    assert torch.equal(reorder_states(x.transpose(0, 1).contiguous().transpose(0, 1), par), x[torch.arange(7, device="cuda")[:, None], par])
    par[2, 1], par[3, 4] = -1, 5  # no beams: the rows stay
    y = reorder_states(x, par)
    assert torch.equal(y[2, 1], x[2, 1]) and torch.equal(y[3, 4], x[3, 4]) and torch.equal(y[0], x[0, par[0]])


# ---- the cache


def both(num_seqs, max_len, heads, dim, layers=1, pages=None):
    """A cache whose memory holds NaN bytes and wild exponents, and its restatement."""
    from asr_amd.decoding import PagedKVCache

    c = PagedKVCache(num_seqs, max_len, heads, dim, num_layers=layers, num_pages=pages)
    c.kv.fill_(0x7F)
    c.exps.fill_(77)
    return c, od.Cache(num_seqs, max_len, heads, dim, layers, pages)


def same_pages(c, o):
    assert np.array_equal(c.table.cpu().numpy(), o.table)
    assert np.array_equal(c.lens.cpu().numpy(), o.lens) and np.array_equal(c.starts.cpu().numpy(), o.starts)
    assert np.array_equal(c.refs.cpu().numpy(), o.refs)
    assert int(c.status[0]) == o.status


def same_tokens(c, o, first, count, every=1):
    view = c if every == 1 else c.leaders(every)
    k, v = view.read(first, count)
    f = first.cpu().numpy() if isinstance(first, torch.Tensor) else first
    for layer in range(o.L):
        for got, want in zip((k, v), o.read(f, count, layer, every)):
            assert np.array_equal(got[layer].double().cpu().numpy(), want, equal_nan=True)
        one = view.read(first, count, layer=layer)
        assert torch.equal(one[0].nan_to_num(9), k[layer].nan_to_num(9)) and torch.equal(one[1].nan_to_num(9), v[layer].nan_to_num(9))


def same_attention(c, o, q, layer=0, beams=1, every=1, scale=None, margins=None, name=""):
    view = c if every == 1 else c.leaders(every)
    got = view.attend(q, layer=layer, num_beams=beams, scale=scale).double().cpu().numpy()
    x = q.double().cpu().numpy()
    want, size = (o.attend(x, layer, scale, every, magnitude=m) for m in (False, True))
    assert np.array_equal(np.isnan(got), np.isnan(want))
    over = np.nan_to_num(np.abs(got - want) / (2.0 ** -8 * np.abs(want) + 2.0 ** -10 * size + 1e-30))
    assert over.max() <= 1, (name, over.max(), np.unravel_index(over.argmax(), over.shape))
    if margins is not None:
        margins.add(f"cache attention {name} vs fp64", over.max(), 1.0, "of the bound")


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 200])
def test_write_and_read(dim, dtype, n):
    c, o = both(5, 500, 3, dim, layers=2)
    g = _gen(n + dim)
    for step, before in enumerate(([0, 0, 0, 0, 0], [1, 63, 64, 37, 0], [0, 5, 0, 64, 130])):  # pages opened at every offset
        c.extend(torch.tensor(before, device="cuda"))
        o.extend(before)
        new = [n, max(0, n - 1), n, 1, (n + 1) // 2]
        for count in (before, new):
            if max(count) == 0:
                continue
            if count is new:
                c.extend(torch.tensor(count, device="cuda", dtype=torch.int32))
                o.extend(count)
            k, v = (torch.randn((5, max(count), 3, dim), generator=g, device="cuda").to(dtype) * 2.0 ** (4 * step) for _ in range(2))
            for layer in (1, 0):
                c.write(k * (1 + layer), v, layer=layer)
                o.write((k * (1 + layer)).double().cpu().numpy(), v.double().cpu().numpy(), layer)
        same_pages(c, o)
        same_tokens(c, o, 0, int(o.lens.max()) + 3)
        same_tokens(c, o, c.starts, 70)
        same_tokens(c, o, torch.tensor([0, 1, 63, 64, 499], device="cuda"), 1)


def test_write_is_right_at_the_ends_of_the_range():
    c, o = both(3, 200, 1, 64)
    rows = torch.zeros((3, 70, 1, 64), device="cuda")
    g = _gen(4)
    rows[0] = torch.randn((70, 1, 64), generator=g, device="cuda") * 2.0 ** torch.randint(-140, 120, (70, 1, 64), generator=g, device="cuda").float()
    rows[1, 0, 0, :8] = torch.tensor([3.4e38, -3.4e38, 1e-45, 1e38, math.inf, -math.inf, math.nan, 0.0])
    rows[1, 64, 0, :4] = torch.tensor([448.0, 449.0, 17.0, 2.0 ** -70])
    rows[2, 3, 0, 0] = 2.0 ** -80  # below the smallest exponent's smallest value
    rows[2, 64, 0, 0] = math.nan
    for n in (1, 5, 64):  # raises the exponents of open pages
        c.extend(n)
        o.extend(n)
        k, v = rows[:, :n], rows[:, 70 - n:]
        c.write(k, v)
        o.write(k.double().cpu().numpy(), v.double().cpu().numpy())
        same_tokens(c, o, 0, 70)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("where", ["keys", "values", "both"])
def test_write_bf16_at_the_ends_of_the_range(dim, where):
    """Pages with and without numbers that are not finite or saturate, in the keys, the values or both."""
    g = _gen(dim)
    c, o = both(3, 200, 2, dim)
    for n in (1, 70, 1, 5, 64):
        k, v = (torch.randn((3, n, 2, dim), generator=g, device="cuda").bfloat16() for _ in range(2))
        for x in {"keys": [k], "values": [v], "both": [k, v]}[where]:
            x[0, n // 2, 0, 3:7] = torch.tensor([math.inf, -math.inf, math.nan, -3e38], device="cuda").bfloat16()
            x[1, n - 1, 1, :2] = torch.tensor([3.3e38, -2.0 ** 127], device="cuda").bfloat16()
            x[2, 0, 0, dim - 1] = -math.nan
        c.extend(n)
        o.extend(n)
        c.write(k, v)
        o.write(k.double().cpu().numpy(), v.double().cpu().numpy())
        same_tokens(c, o, 0, 200)


def test_write_takes_any_strides():
    c, o = both(2, 130, 2, 64)
    g = _gen(8)
    fused = torch.randn((2, 66, 8, 64), generator=g, device="cuda").bfloat16()
    for k, v in ((fused[:, :, 4:6], fused[:, :, 6:]), (fused[:, :, 1:6:3], fused[:, :, 2:4]), (fused[:, :, :2].transpose(1, 2).contiguous().transpose(1, 2), fused[:, :, 6:]),
                 (fused.view(-1)[1:1 + 66 * 2 * 64 * 2].view(2, 66, 2, 64), fused[:, :, 6:]), (fused[:1, :, :2].expand(2, 66, 2, 64), fused[:1, :, 2:4].expand(2, 66, 2, 64))):
        c.reorder(torch.full((1, 2), -1, device="cuda"))
        o.reorder([[-1, -1]])
        c.extend(66)
        o.extend(66)
        c.write(k, v)
        o.write(k.double().cpu().numpy(), v.double().cpu().numpy())
        same_tokens(c, o, 0, 66)


@pytest.mark.parametrize("seed", range(4))
def test_pages_over_a_random_life(seed):
    """Prompts enter, are forked, grow, end and are compacted, in a pool that now and then is too small."""
    rng = np.random.default_rng(seed)
    B, K = [(2, 3), (3, 1), (1, 5), (4, 2)][seed]
    c, o = both(B * K, 330, 2, 64, layers=2, pages=[16, 9, 14, 40][seed])
    lead = c.leaders(K)

    def put(cache, n, every):  # every token is written, in both layers
        cache.extend(torch.from_numpy(n).cuda())
        o.extend(n, every)
        for layer in range(2):
            k, v = (torch.from_numpy(rng.standard_normal((len(n), int(n.max()), 2, 64)) * 2.0 ** rng.integers(-3, 4)).float().cuda() for _ in range(2))
            cache.write(k, v, layer=layer)
            o.write(k.double().cpu().numpy(), v.double().cpu().numpy(), layer, every)

    for step in range(40):
        what = rng.integers(0, 6)
        if what == 0:
            put(lead, rng.integers(0, 150, B), K)
        elif what == 1:
            par = rng.integers(0, K, (B, K))
            c.reorder(torch.from_numpy(par).cuda())
            o.reorder(par)
        elif what == 2:
            par = np.where(rng.random((B, K)) < 0.4, -1, np.arange(K))
            c.reorder(torch.from_numpy(par).cuda())
            o.reorder(par)
        elif what == 3:
            used = c.compact()
            assert int(used) == o.compact()
        elif what == 4:
            put(c, np.full(B * K, rng.integers(1, 70)), 1)
        else:
            put(c, rng.integers(0, 3, B * K), 1)
        same_pages(c, o)
        same_tokens(c, o, 0, 330)


def test_pages_of_thousands_of_sequences():
    """More sequences than threads in the workgroup that hands out pages, and more pages than it looks at in one go."""
    rng = np.random.default_rng(77)
    B, K = 700, 3
    c, o = both(B * K, 192, 1, 64, pages=20000)
    lead = c.leaders(K)
    for n in (rng.integers(0, 100, B), rng.integers(0, 3, B)):
        lead.extend(torch.from_numpy(n).cuda())
        o.extend(n, K)
        same_pages(c, o)
    for _ in range(3):
        par = rng.integers(0, K, (B, K)) * (rng.random((B, 1)) < 0.7)
        par = np.where(rng.random((B, K)) < 0.1, -1, par)
        c.reorder(torch.from_numpy(par).cuda())
        o.reorder(par)
        n = rng.integers(0, 30, B * K)
        c.extend(torch.from_numpy(n).cuda())
        o.extend(n)
        same_pages(c, o)
        assert int(c.compact()) == o.compact()
        same_pages(c, o)
    assert o.status in (0, 2)


@pytest.mark.parametrize("B,K", [(32, 32), (41, 25), (512, 2), (128, 8), (1000, 1), (3, 17)])
@pytest.mark.parametrize("pages", [700, 2500, 9000])
def test_pages_shared_by_many(B, K, pages):
    """About as many sequences as the workgroup has threads, pages with up to 32 holders of which all, some or one write, and
    steps that hand out more pages than the workgroup has threads."""
    rng = np.random.default_rng(1000 * pages + 10 * B + K)
    c, o = both(B * K, 320, 1, 64, pages=pages)
    lead = c.leaders(K)
    n = rng.integers(0, 130, B)
    lead.extend(torch.from_numpy(n).cuda())
    o.extend(n, K)
    same_pages(c, o)
    for step in range(4):
        par = np.zeros((B, K), np.int64) if step == 0 else rng.integers(-1, K, (B, K))
        c.reorder(torch.from_numpy(par).cuda())
        o.reorder(par)
        same_pages(c, o)
        for n in (rng.integers(0, 2, B * K), np.ones(B * K, np.int64), rng.integers(0, 100, B * K)):
            c.extend(torch.from_numpy(n).cuda())
            o.extend(n)
            same_pages(c, o)


def test_what_does_not_fit_adds_nothing_and_is_reported():
    from asr_amd import _lib

    c, o = both(4, 256, 1, 64, pages=5)
    c.extend(70)  # 8 pages
    o.extend(70)
    same_pages(c, o)
    with pytest.raises(_lib.AsrkError, match="pages"):
        c.check()
    c.check()
    o.status = 0
    for n in ([64, 64, 64, 64], [1, 0, 0, 0], [1, 1, 0, 0], [200, 0, 0, 0], [-1, 0, 0, 0]):
        c.extend(torch.tensor(n, device="cuda"))
        o.extend(n)
        same_pages(c, o)
    with pytest.raises(_lib.AsrkError, match="pages.*max_len.*negative"):
        c.check()
    o.status = 0
    c.reorder(torch.tensor([[1, 4], [-2, 0]], device="cuda"))
    o.reorder([[1, 4], [-2, 0]])
    same_pages(c, o)
    with pytest.raises(_lib.AsrkError, match="parent"):
        c.check()
    k = torch.ones((4, 3, 1, 64), device="cuda")
    c.write(k, k)  # no row is new
    assert int((c.kv != 0x7F).sum()) == 0 and int((c.attend(k.bfloat16()) != 0).sum()) == 0


def filled(rng, num_seqs, heads, dim, before, new, beams=1, shared=None, layers=1):
    """Sequences of `before` tokens and `new` ones in both caches; groups of `beams` share their first `shared` tokens."""
    before, new = np.asarray(before), np.asarray(new)
    top = int((before + new).max()) + 1
    c, o = both(num_seqs, top, heads, dim, layers, pages=num_seqs * (-(-top // 64)) + 3)
    lead = c.leaders(beams)

    def put(x, cache, every, n):
        rows = int(max(n))
        if rows == 0:
            return
        k, v = (torch.from_numpy(rng.standard_normal((len(n), rows, heads, dim)) * s).float().cuda() for s in (1.0, 1.5))
        for layer in range(layers):
            cache.write(k, v, layer=layer)
            o.write(k.double().cpu().numpy(), v.double().cpu().numpy(), layer, every)

    if beams > 1:
        first = np.minimum(shared, before[::beams])
        lead.extend(torch.from_numpy(first).cuda())
        o.extend(first, beams)
        put(None, lead, beams, first)
        zero = np.zeros((num_seqs // beams, beams), np.int64)
        c.reorder(torch.from_numpy(zero).cuda())
        o.reorder(zero)
        rest = before - np.repeat(first, beams)
    else:
        rest = before
    for n in (rest, new):
        c.extend(torch.from_numpy(n).cuda())
        o.extend(n)
        put(None, c, 1, n)
    same_pages(c, o)
    c.check()
    return c, o


@pytest.mark.parametrize("dim,heads,group", [(64, 5, 3), (64, 1, 8), (64, 2, 1), (128, 2, 4), (128, 1, 16), (128, 3, 7)])
def test_attend_single_tokens(dim, heads, group, margins):
    rng = np.random.default_rng(dim + group)
    before = [0, 1, 62, 63, 64, 127, 300, 700]
    c, o = filled(rng, 8, heads, dim, before, [1, 1, 1, 1, 1, 0, 1, 1])  # sequence 5 has ended
    q = torch.from_numpy(rng.standard_normal((8, 1, heads * group, dim))).cuda().bfloat16() * 2
    same_attention(c, o, q, margins=margins, name=f"1 token, d {dim}, {heads} x {group}")
    assert int((c.attend(q)[5] != 0).sum()) == 0


@pytest.mark.parametrize("dim,heads,group,n", [(64, 5, 3, 2), (64, 1, 1, 70), (128, 2, 2, 9), (64, 2, 3, 130), (128, 1, 4, 200), (128, 1, 17, 8), (64, 1, 128, 1)])
def test_attend_several_tokens(dim, heads, group, n, margins):
    """Prompts behind what is there: every row sees the tokens up to its own; short sequences leave rows empty."""
    rng = np.random.default_rng(n)
    c, o = filled(rng, 4, heads, dim, [0, 5, 64, 130], [n, max(0, n - 1), (n + 1) // 2, 0])
    q = torch.from_numpy(rng.standard_normal((4, n, heads * group, dim))).cuda().bfloat16()
    same_attention(c, o, q, margins=margins, name=f"{n} tokens, d {dim}, {heads} x {group}")
    same_attention(c, o, q, scale=0.5, name="another scale")


@pytest.mark.parametrize("dim,heads,group,beams,n", [(64, 5, 3, 5, 1), (128, 1, 4, 4, 1), (64, 1, 1, 32, 1), (64, 2, 2, 3, 3), (128, 2, 7, 5, 1), (64, 1, 8, 8, 2), (64, 1, 16, 4, 3), (128, 1, 16, 5, 4)])
def test_attend_beams(dim, heads, group, beams, n, margins):
    """Beams that share all pages but the last, some, or none; num_beams says which are worked on together and nothing else."""
    rng = np.random.default_rng(beams)
    S = 3 * beams
    before = np.repeat([260, 129, 64], beams) + rng.integers(0, 70, S) * np.repeat([0, 1, 0], beams)
    new = rng.integers(0, n + 1, S)
    new[:beams] = n
    c, o = filled(rng, S, heads, dim, before, new, beams, np.array([250, 70, 64]))
    q = torch.from_numpy(rng.standard_normal((S, n, heads * group, dim))).cuda().bfloat16()
    same_attention(c, o, q, beams=beams, margins=margins, name=f"{beams} beams, d {dim}, {heads} x {group}, {n} tokens")
    same_attention(c, o, q, beams=1, name="apart")
    if beams * n * group <= 16:  # the same kernel: a row's bits do not depend on the rows that it is worked on with
        assert torch.equal(c.attend(q, num_beams=beams), c.attend(q))
    par = rng.integers(0, beams, (3, beams))  # pages shared in no order
    c.reorder(torch.from_numpy(par).cuda())
    o.reorder(par)
    assert int((c.attend(q, num_beams=beams) != 0).sum()) == 0  # nothing is new
    new = np.minimum(n, rng.integers(0, 2 * n + 1, S))
    c.extend(torch.from_numpy(new).cuda())
    o.extend(new)
    k, v = (torch.from_numpy(rng.standard_normal((S, n, heads, dim))).float().cuda() for _ in range(2))
    c.write(k, v)
    o.write(k.double().cpu().numpy(), v.double().cpu().numpy())
    same_attention(c, o, q, beams=beams, name="reordered")


@pytest.mark.parametrize("beams", [1, 3])
@pytest.mark.parametrize("n", [1, 40])
def test_attend_keeps_nan_where_it_is_seen(beams, n):
    """A NaN reaches the rows that see its token, and no others: not the earlier rows, not the other beams, not past the end."""
    rng = np.random.default_rng(7)
    S = 2 * beams
    c, o = filled(rng, S, 1, 64, [100] * S, [n] * S, beams, np.array([90, 64]))
    k, v = (torch.from_numpy(rng.standard_normal((S, n, 1, 64))).float().cuda() for _ in range(2))
    v[1, n // 2, 0, 5] = math.inf
    v[0, n - 1, 0, 63] = math.nan
    k[S - 1, n - 1, 0, 0] = math.nan
    c.write(k, v)
    o.write(k.double().cpu().numpy(), v.double().cpu().numpy())
    q = torch.from_numpy(rng.standard_normal((S, n, 3, 64))).cuda().bfloat16()
    same_attention(c, o, q, beams=beams)
    assert bool(c.attend(q, num_beams=beams).isnan().any()) and not bool(c.attend(q, num_beams=beams).isnan().all())


def test_attend_over_pages_of_very_different_scales():
    """Values of 2**-60 next to values of 2**60: each row is right to its own size where the weights say so."""
    rng = np.random.default_rng(9)
    c, o = both(2, 320, 1, 64)
    for e in (-50.0, 3.0, -9.0, 60.0):
        c.extend(64)
        o.extend(64)
        k = torch.from_numpy(rng.standard_normal((2, 64, 1, 64))).float().cuda()
        v = torch.from_numpy(rng.standard_normal((2, 64, 1, 64))).float().cuda() * 2.0 ** e
        c.write(k, v)
        o.write(k.double().cpu().numpy(), v.double().cpu().numpy())
        q = torch.from_numpy(rng.standard_normal((2, 64, 2, 64))).cuda().bfloat16()
        same_attention(c, o, q)
        same_attention(c, o, q[:, :1])


@pytest.mark.parametrize("beams,n,group", [(1, 1, 2), (1, 8, 4), (1, 40, 4), (3, 1, 4), (2, 20, 4)])
@pytest.mark.parametrize("dim", [64, 128])
def test_attend_splits_long_caches(dim, beams, n, group, margins):
    """Over 48 pages the tokens are split over workgroups and joined, for few columns and for many."""
    rng = np.random.default_rng(beams + n)
    S = 2 * beams
    c, o = filled(rng, S, 1, dim, [3300, 64 * 40][:1] * beams + [64 * 40] * beams, [n] * S, beams, np.array([3200, 64 * 39]))
    q = torch.from_numpy(rng.standard_normal((S, n, group, dim))).cuda().bfloat16()
    same_attention(c, o, q, beams=beams, margins=margins, name=f"3300 tokens, {beams} beams, {n} tokens, d {dim}")


def test_attend_over_many_sequences():
    """More workgroups than a grid's second and third dimensions hold."""
    S, n, group = 9000, 100, 16
    c, o = both(S, 110, 1, 64)
    g = _gen(91)
    for rows in (7, n):
        c.extend(rows)
        o.extend(rows)
        k, v = (torch.randn((S, rows, 1, 64), generator=g, device="cuda").bfloat16() for _ in range(2))
        c.write(k, v)
        o.write(k[::3000].double().cpu().numpy(), v[::3000].double().cpu().numpy(), every=3000)
    q = torch.randn((S, n, group, 64), generator=g, device="cuda").bfloat16()
    got = c.attend(q)[::3000]
    assert torch.equal(got, c.leaders(3000).attend(q[::3000]))
    same_attention(c, o, q[::3000, :, :2], every=3000)


@pytest.mark.parametrize("n", [1, 130])
@pytest.mark.parametrize("low", [8.0, 14.2, 17.3, 20.0])
def test_attend_adds_up_many_small_weights(n, low):
    """One token that outweighs each of 20000 others by 2**(low * 1.44): what they add up to is the result, to its own size (and
    half a step of 2**-37, times the largest weight, for each of them: weights below 2**-27 of the largest are subnormal)."""
    c = PagedKVCache_(1, 20300, 1, 64)
    k, v = (torch.zeros((1, 20000, 1, 64), device="cuda") for _ in range(2))
    k[:, 0, :, 0] = 2.0 ** round(math.log2(low))
    v[:, 1:] = 1.0
    c.extend(20000)
    c.write(k, v)
    c.extend(n)
    c.write(torch.zeros((1, n, 1, 64), device="cuda"), torch.ones((1, n, 1, 64), device="cuda"))
    q = torch.zeros((1, n, 1, 64), device="cuda", dtype=torch.bfloat16)
    top = float(torch.tensor(low * 8 / 2.0 ** round(math.log2(low))).bfloat16())  # q.k / 8 is about low
    q[..., 0] = top
    s = top * 2.0 ** round(math.log2(low)) / 8
    got = c.attend(q).double().cpu().numpy()
    others = 20000 + np.arange(n).reshape(1, n, 1, 1)  # tokens of weight exp(-s) and value 1
    want = others * math.exp(-s) / (1 + others * math.exp(-s))
    over = np.abs(got - want) / (want * (2.0 ** -8 + 2.0 ** -10) + others * 2.0 ** -38)
    assert over.max() <= 1, over.max()


def test_a_write_after_reorder_waits_for_extend():
    """Beams that have just come to share a page do not write into it."""
    rng = np.random.default_rng(5)
    c, o = filled(rng, 3, 1, 64, [70, 70, 70], [1, 1, 1], 3, np.array([60]))
    par = np.array([[1, 1, 1]])
    c.reorder(torch.from_numpy(par).cuda())
    o.reorder(par)
    before = c.kv.clone(), c.exps.clone()
    k, v = (torch.randn((3, 1, 1, 64), device="cuda") * 100 for _ in range(2))
    c.write(k, v)
    assert torch.equal(c.kv, before[0]) and torch.equal(c.exps, before[1])
    c.extend(1)
    o.extend(1)
    c.write(k, v)
    o.write(k.double().cpu().numpy(), v.double().cpu().numpy())
    same_pages(c, o)
    same_tokens(c, o, 0, 80)


@pytest.mark.parametrize("gap", [16, 30, 60])
@pytest.mark.parametrize("n,group", [(1, 3), (1, 20), (50, 2)])
def test_attend_beams_of_very_different_scales(gap, n, group):
    """Beams whose values are 2**gap apart do not cost each other bits, whichever comes first."""
    rng = np.random.default_rng(gap)
    S = 4
    c, o = both(S, 300, 1, 64)
    for rows in (130, n):
        c.extend(rows)
        o.extend(rows)
        k, v = (torch.from_numpy(rng.standard_normal((S, rows, 1, 64))).float().cuda() for _ in range(2))
        v *= torch.tensor([0, gap, -gap / 2, 3], device="cuda").exp2().view(S, 1, 1, 1)
        c.write(k, v)
        o.write(k.double().cpu().numpy(), v.double().cpu().numpy())
    q = torch.from_numpy(rng.standard_normal((S, n, group, 64))).cuda().bfloat16()
    same_attention(c, o, q, beams=S)
    same_attention(c, o, q, beams=2)


@pytest.mark.parametrize("n,max_len", [(1, 300), (1, 4000), (100, 300), (100, 4000)])
def test_attend_at_the_end_of_the_range(n, max_len):
    """Values up to 2**127: sums of weighted values would overflow, their averages do not."""
    rng = np.random.default_rng(n)
    c, o = both(2, max_len, 1, 64)
    for rows in (130, n):
        c.extend(rows)
        o.extend(rows)
        k, v = (torch.from_numpy(rng.standard_normal((2, rows, 1, 64))).float().cuda() for _ in range(2))
        v = v.clamp(-3, 3) * torch.tensor([2.0 ** 125, 2.0 ** 100], device="cuda").view(2, 1, 1, 1)
        c.write(k, v)
        o.write(k.double().cpu().numpy(), v.double().cpu().numpy())
    q = torch.from_numpy(rng.standard_normal((2, n, 2, 64))).cuda().bfloat16()
    same_attention(c, o, q)
    same_attention(c, o, q, beams=2)


@pytest.mark.parametrize("power", [16, 30, 100])
@pytest.mark.parametrize("n,max_len", [(1, 300), (1, 4000), (100, 300), (100, 4000)])
def test_attend_with_enormous_scores(n, max_len, power):
    """Scores whose neighbouring fp32 numbers lie far apart: the largest wins, and equal ones share.  Keys of +-2**power and
    small integers in q, so that every score is exact and ties are ties."""
    rng = np.random.default_rng(n + power)
    c, o = both(3, max_len, 1, 64)
    for rows in (130, n):
        c.extend(rows)
        o.extend(rows)
        k, v = (torch.from_numpy(x).float().cuda() for x in (rng.choice([-1.0, 1.0], (3, rows, 1, 64)) * 2.0 ** power, rng.standard_normal((3, rows, 1, 64))))
        c.write(k, v)
        o.write(k.double().cpu().numpy(), v.double().cpu().numpy())
    q = torch.from_numpy(rng.integers(-3, 4, (3, n, 2, 64))).cuda().bfloat16()
    q[1, :, 1] *= 2.0 ** -power  # beside ordinary ones
    q[2, :, 0] = 1
    same_attention(c, o, q)
    same_attention(c, o, q, beams=3)


@pytest.mark.parametrize("n", [1, 100])
def test_attend_keeps_the_queries_nan(n):
    """A query with a NaN or an infinity gives NaN, and changes no other row."""
    rng = np.random.default_rng(n)
    c, o = filled(rng, 2, 1, 64, [130, 200], [n, n])
    q = torch.from_numpy(rng.standard_normal((2, n, 3, 64))).cuda().bfloat16()
    clean = c.attend(q)
    q[0, n // 2, 1, 5], q[1, n - 1, 0, 9], q[1, 0, 2, 60] = float("nan"), float("inf"), float("-inf")
    with np.errstate(invalid="ignore"):
        same_attention(c, o, q)
    got = c.attend(q)
    hit = torch.isnan(q).any(-1) | torch.isinf(q).any(-1)
    assert bool(got[hit].isnan().all()) and torch.equal(got[~hit], clean[~hit])


def test_attend_refuses_more_rows_than_one_call_takes():
    c, _ = both(1, 64, 1, 64)
    q = torch.zeros((1, 1, 4, 64), device="cuda", dtype=torch.bfloat16).expand(1, 65535 * 128 // 4 + 1, 4, 64)
    with pytest.raises(ValueError, match="one call"):
        c.attend(q)


def test_attend_takes_any_strides():
    rng = np.random.default_rng(10)
    c, o = filled(rng, 3, 2, 64, [70, 3, 100], [2, 2, 2], layers=2)
    fused = torch.from_numpy(rng.standard_normal((3, 5, 14, 64))).cuda().bfloat16()
    for q in (fused[:, :2, :6], fused[:, 3:, 8:], fused[:, ::4, 1:13:2], fused.transpose(1, 2)[:, 4:6, :4].contiguous(), fused.view(-1)[3:3 + 3 * 2 * 4 * 64].view(3, 2, 4, 64),
              fused[:1, :2, :4].expand(3, 2, 4, 64)):
        same_attention(c, o, q, layer=1)


def test_leaders_view_reads_and_attends():
    rng = np.random.default_rng(12)
    c, o = filled(rng, 6, 1, 128, [40, 9, 9, 90, 9, 9], [3, 1, 1, 3, 1, 1])
    q = torch.from_numpy(rng.standard_normal((2, 3, 2, 128))).cuda().bfloat16()
    same_attention(c, o, q, every=3)
    same_tokens(c, o, 30, 70, every=3)


def test_offsets_pass_32_bits():
    """Two layers of 300000 pages of 16 KiB: the pages in use lie beyond 8 GiB."""
    from asr_amd.decoding import PagedKVCache

    P = 300000
    c = PagedKVCache(2, 256, 1, 128, num_layers=2, num_pages=P)
    o = od.Cache(2, 256, 1, 128, 2, 8)
    c.refs[:P - 8] = 1  # held by others
    c.extend(130)
    o.extend(130)
    assert np.array_equal(c.table.cpu().numpy(), np.where(o.table >= 0, o.table + P - 8, -1))
    g = _gen(2)
    k, v = (torch.randn((2, 130, 1, 128), generator=g, device="cuda") for _ in range(2))
    c.write(k, v, layer=1)
    o.write(k.double().cpu().numpy(), v.double().cpu().numpy(), 1)
    same_tokens(c, o, 0, 140)
    same_attention(c, o, torch.randn((2, 1, 4, 128), generator=g, device="cuda").bfloat16(), layer=1)
    c.refs[:P - 8] = 0
    assert int(c.compact()) == 6 and int(c.table.max()) == 5
    same_tokens(c, o, 0, 140)


def test_refusals():
    from asr_amd import _lib
    from asr_amd.decoding import PagedKVCache, beam_select, reorder_states

    c = PagedKVCache(4, 100, 2, 64, num_layers=2)
    ok = torch.zeros((4, 1, 2, 64), device="cuda", dtype=torch.bfloat16)
    for k, v in ((ok[:3], ok[:3]), (ok, ok[:, :, :1]), (ok.half(), ok.half()), (ok, ok.float()), (ok[0], ok[0]), (ok[..., :32], ok[..., :32])):
        with pytest.raises(ValueError):
            c.write(k, v)
    for q, kw in ((ok[:3], {}), (ok.float(), {}), (ok[:, :, :1], {}), (ok[..., :32], {}), (ok, dict(num_beams=3)), (ok, dict(num_beams=0)), (ok, dict(layer=2)),
                  (ok, dict(layer=-1)), (ok[:, :, :0], {}), (ok, dict(scale=0.0)), (ok, dict(scale=-1.0)), (ok, dict(scale=math.nan)), (ok, dict(scale=math.inf))):
        with pytest.raises(ValueError):
            c.attend(q, **kw)
    with pytest.raises(ValueError):
        c.attend(ok.clone().requires_grad_())
    with pytest.raises(ValueError):
        beam_select(torch.zeros((4, 9), device="cuda", requires_grad=True), torch.zeros((2, 2), device="cuda"))
    for n in (-1, 129, torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(4, device="cuda"), torch.zeros((4, 1), dtype=torch.int32, device="cuda")):
        with pytest.raises(ValueError):
            c.extend(n)
    for p in (torch.zeros((2, 2), dtype=torch.int32, device="cuda"), torch.zeros((2, 3), dtype=torch.int64, device="cuda"), torch.zeros((4,), dtype=torch.int64, device="cuda")):
        with pytest.raises(ValueError):
            c.reorder(p)
    for bad in (lambda: c.read(-1, 3), lambda: c.read(0, -1), lambda: c.read(0, 3, layer=2), lambda: c.read(torch.zeros(3, dtype=torch.int32, device="cuda"), 3),
                lambda: c.leaders(3), lambda: c.leaders(0), lambda: c.leaders(2).compact()):
        with pytest.raises(ValueError):
            bad()
    for cpu in (lambda: c.write(ok.cpu(), ok.cpu()), lambda: c.attend(ok.cpu()), lambda: c.extend(torch.zeros(4, dtype=torch.int32)), lambda: c.reorder(torch.zeros((2, 2), dtype=torch.int64))):
        with pytest.raises(_lib.AsrkError):
            cpu()
    with pytest.raises(ValueError):
        reorder_states(ok.cpu(), torch.zeros((2, 2), dtype=torch.int64, device="cuda")) if False else reorder_states(ok[:3], torch.zeros((2, 2), dtype=torch.int64, device="cuda"))
    assert tuple(c.attend(ok[:, :0]).shape) == (4, 0, 2, 64)
    c.write(ok[:, :0], ok[:, :0])
    assert tuple(c.read(0, 0)[0].shape) == (2, 4, 0, 2, 64)
    assert beam_select(torch.zeros((0, 9), device="cuda"), torch.zeros((0, 2), device="cuda")).tokens.shape == (0, 2)
    assert int(c.status[0]) == 0 and int(c.lens.sum()) == 0


# ---- together


def _step(c, logits, scores, history, k, v, q, beams, eos):
    from asr_amd.decoding import beam_select, reorder_states

    step = beam_select(logits, scores, eos)
    c.reorder(step.parents)
    history.copy_(reorder_states(history, step.parents))
    c.extend(1)
    for layer in range(c.num_layers):
        c.write(k[layer], v[layer], layer=layer)
    out = torch.stack([c.attend(q[layer], layer=layer, num_beams=beams) for layer in range(c.num_layers)])
    scores.copy_(step.scores)
    return out, step.tokens


def _prompted(seed, B, K, heads, dim, layers, prompt, max_len):
    from asr_amd.decoding import PagedKVCache

    g = _gen(seed)
    c = PagedKVCache(B * K, max_len, heads, dim, num_layers=layers)
    lead = c.leaders(K)
    lead.extend(torch.tensor([prompt - i for i in range(B)], device="cuda"))
    for layer in range(layers):
        k, v = (torch.randn((B, prompt, heads, dim), generator=g, device="cuda").bfloat16() for _ in range(2))
        lead.write(k, v, layer=layer)
    c.reorder(torch.zeros((B, K), dtype=torch.int64, device="cuda"))
    return c


def _inputs(seed, B, K, heads, group, dim, layers, V):
    g = _gen(seed)
    return dict(logits=torch.randn((B * K, V), generator=g, device="cuda") * 3,
                k=torch.randn((layers, B * K, 1, heads, dim), generator=g, device="cuda").bfloat16(),
                v=torch.randn((layers, B * K, 1, heads, dim), generator=g, device="cuda").bfloat16(),
                q=torch.randn((layers, B * K, 1, heads * group, dim), generator=g, device="cuda").bfloat16())


def test_steps_together_follow_the_oracle():
    B, K, heads, group, dim, V = 2, 3, 2, 2, 64, 57
    c, o = both(B * K, 200, heads, dim)
    rng = np.random.default_rng(21)
    n = np.array([70, 61])
    c.leaders(K).extend(torch.from_numpy(n).cuda())
    o.extend(n, K)
    k, v = (torch.from_numpy(rng.standard_normal((B, 70, heads, dim))).float().cuda() for _ in range(2))
    c.leaders(K).write(k, v)
    o.write(k.double().cpu().numpy(), v.double().cpu().numpy(), every=K)
    zero = np.zeros((B, K), np.int64)
    c.reorder(torch.from_numpy(zero).cuda())
    o.reorder(zero)
    scores = torch.zeros((B, K), device="cuda")
    scores[:, 1:] = -math.inf
    for t in range(12):
        x = _inputs(100 + t, B, K, heads, group, dim, 1, V)
        step = check_select(x["logits"], scores, eos=5)
        c.reorder(step.parents)
        o.reorder(step.parents.cpu().numpy())
        c.extend(1)
        o.extend(1)
        c.write(x["k"][0], x["v"][0])
        o.write(x["k"][0].double().cpu().numpy(), x["v"][0].double().cpu().numpy())
        same_pages(c, o)
        same_attention(c, o, x["q"][0], beams=K)
        scores = step.scores
    same_tokens(c, o, 0, 90)


def test_a_captured_step_replays_like_the_eager_one():
    B, K, heads, group, dim, layers, V = 2, 4, 2, 3, 64, 2, 4099
    args = (31, B, K, heads, dim, layers, 90, 200)
    eager, graphed = _prompted(*args), _prompted(*args)
    state = {}
    for name in ("eager", "graphed"):
        s = torch.zeros((B, K), device="cuda")
        s[:, 1:] = -math.inf
        state[name] = dict(scores=s, history=torch.arange(B * K * 7, device="cuda").view(B, K, 7))
    x = _inputs(1, B, K, heads, group, dim, layers, V)
    warm = _prompted(*args)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        _step(warm, **{n: t.clone() for n, t in x.items()}, beams=K, eos=7, **{n: t.clone() for n, t in state["eager"].items()})
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = _step(graphed, **x, beams=K, eos=7, **state["graphed"])
    for t in range(80):  # over the end of a page and of max_len's table
        fresh = _inputs(200 + t, B, K, heads, group, dim, layers, V)
        for n, tensor in fresh.items():
            x[n].copy_(tensor)
        graph.replay()
        want = _step(eager, **fresh, beams=K, eos=7, **state["eager"])
        if t % 9 == 0:
            torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), t
        for n in ("table", "lens", "starts", "refs", "kv", "exps"):
            assert torch.equal(getattr(eager, n), getattr(graphed, n)), (t, n)
        assert torch.equal(state["eager"]["scores"], state["graphed"]["scores"]) and torch.equal(state["eager"]["history"], state["graphed"]["history"])
    assert int(eager.lens.max()) == 170
    eager.check()


def test_two_caches_on_two_streams():
    args = (41, 2, 5, 1, 64, 1, 130, 300)
    want = _prompted(*args)
    outs = []
    streams = [torch.cuda.Stream() for _ in range(2)]
    caches = [_prompted(*args) for _ in range(2)]
    torch.cuda.synchronize()
    scores = [torch.zeros((2, 5), device="cuda") for _ in range(3)]
    hist = [torch.zeros((2, 5, 3), device="cuda", dtype=torch.int64) for _ in range(3)]
    xs = [_inputs(300 + t, 2, 5, 1, 3, 64, 1, 9001) for t in range(10)]
    torch.cuda.synchronize()
    for t in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs.append(_step(caches[i], **xs[t], beams=5, eos=3, scores=scores[i], history=hist[i])[0])
    ref = [_step(want, **xs[t], beams=5, eos=3, scores=scores[2], history=hist[2])[0] for t in range(10)]
    torch.cuda.synchronize()
    for t in range(10):
        assert torch.equal(outs[2 * t], ref[t]) and torch.equal(outs[2 * t + 1], ref[t])


class TinyDecoder:
    """One layer: attention over the cache and a residual, to logits."""

    num_layers, kv_heads, head_dim, group = 1, 2, 64, 2

    def __init__(self, vocab, width=48, seed=0):
        g = _gen(seed)
        r = lambda *shape: torch.randn(shape, generator=g, device="cuda") / math.sqrt(shape[0])  # noqa: E731
        heads, d = self.kv_heads * self.group, self.head_dim
        self.emb, self.wq, self.wk, self.wv = r(vocab, width) * 7, r(width, heads * d), r(width, self.kv_heads * d), r(width, self.kv_heads * d)
        self.wo, self.wx = r(heads * d, vocab) * 6, r(width, vocab) * 3

    def embed(self, tokens):
        return self.emb[tokens]

    def qkv(self, x):
        S, n, _ = x.shape
        return ((x @ w).bfloat16().view(S, n, -1, self.head_dim) for w in (self.wq, self.wk, self.wv))

    def __call__(self, x, cache, num_beams):
        q, k, v = self.qkv(x)
        cache.write(k, v)
        o = cache.attend(q, num_beams=num_beams).double()
        y = o.flatten(2) @ self.wo.double() + x.double() @ self.wx.double()
        last = (cache.lens - cache.starts).long() - 1
        return y[torch.arange(len(y), device="cuda"), last].float()


def plain_beam_search(dec, embeds, lens, K, steps, eos, penalty):
    """One utterance at a time: hypotheses in Python lists, the oracle's selection, and a cache of its own for every beam, which
    is copied whole when a beam continues another (no page is shared, nothing is reordered)."""
    from asr_amd.decoding import PagedKVCache

    def copied(c):
        new = PagedKVCache(1, c.max_len, dec.kv_heads, dec.head_dim)
        for name in ("kv", "exps", "table", "lens", "starts", "refs"):
            getattr(new, name).copy_(getattr(c, name))
        return new

    out = []
    for b in range(len(lens)):
        caches = [PagedKVCache(1, int(lens[b]) + steps, dec.kv_heads, dec.head_dim)]
        caches[0].extend(int(lens[b]))
        logits = dec(embeds[b:b + 1, :lens[b]], caches[0], 1).expand(K, -1)
        caches, scores, beams, ended, done = caches * K, np.array([[0.0] + [-np.inf] * (K - 1)]), [[]] * K, [], False
        for t in range(steps):
            s, tok, par, cs, ct, cp = od.select(logits.double().cpu().numpy()[None], scores, eos)
            for j in range(K):
                if ct[0, j] == eos and not done:
                    ended.append((cs[0, j] / (t + 1) ** penalty, beams[cp[0, j]]))
            ended = sorted(ended, key=lambda e: -e[0])[:K]
            done = done or (len(ended) == K and s[0, 0] / (t + 1) ** penalty <= ended[-1][0])
            beams = [beams[par[0, j]] + [int(tok[0, j])] for j in range(K)]
            scores = s
            if t + 1 == steps or done:
                break
            caches = [copied(caches[par[0, j]]) for j in range(K)]
            for c in caches:
                c.extend(1)
            logits = torch.cat([dec(dec.embed(torch.tensor([[tok[0, j]]], device="cuda")), c, 1) for j, c in enumerate(caches)])
        if not done:
            ended += [(scores[0, j] / (t + 1) ** penalty, beams[j]) for j in range(K)]
        best = max(ended, key=lambda e: e[0])
        out.append((best[1], best[0]))
    return out


@pytest.mark.parametrize("K,penalty,steps", [(1, 1.0, 20), (3, 1.0, 40), (5, 0.0, 30), (4, 2.0, 70)])
def test_beam_generate_follows_a_plain_beam_search(K, penalty, steps):
    from asr_amd.evaluation import beam_generate

    dec = TinyDecoder(37, seed=K)
    embeds = torch.randn((3, 90, 48), generator=_gen(50 + K), device="cuda")
    lens = torch.tensor([90, 13, 64], device="cuda")
    tokens, scores = beam_generate(dec, embeds, num_beams=K, max_new_tokens=steps, eos_token_id=4, length_penalty=penalty, prompt_lens=lens)
    for b, (want, score) in enumerate(plain_beam_search(dec, embeds, lens.tolist(), K, steps, 4, penalty)):
        assert tokens[b] == want, (b, tokens[b], want)
        assert abs(float(scores[b]) - score) <= 1e-5 * steps  # float32 logits and scores in every step
    assert any(len(t) < steps for t in tokens) or K == 1


def test_beam_generate_refusals():
    from asr_amd.evaluation import beam_generate

    dec, x = TinyDecoder(9), torch.zeros((2, 5, 48), device="cuda")
    for kw in (dict(max_new_tokens=0), dict(check_every=0), dict(num_beams=17), dict(prompt_lens=torch.tensor([1, 6], device="cuda")),
               dict(prompt_lens=torch.tensor([0, 2], device="cuda"))):
        with pytest.raises(ValueError):
            beam_generate(dec, x, **kw)
    with pytest.raises(ValueError):
        beam_generate(dec, x[0])
    tokens, scores = beam_generate(dec, x, num_beams=2, max_new_tokens=3)  # no end token
    assert [len(t) for t in tokens] == [3, 3] and bool(scores.isfinite().all())
