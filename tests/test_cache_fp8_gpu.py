"""The kernels of a cache in 8 bits against tests/fp8_cache.py: what an append leaves, bit for bit, and attention against
64-bit arithmetic over what the cache holds.

Bounds on attention. The kernels read exact numbers (codes, exponents, bfloat16 queries); what they round is the weights
(the tensor-core kernels: half precision, 2^-11 relative), the exponentials (2^-21 relative, and an argument of up to 2^7 in
units of log2 that carries 2^-24 of itself, 2^-17), sums over up to 2^11 keys in float32 (2^-24 a step, 2^-13 together at
worst) and the output (bfloat16: 2^-8; float32: 2^-24). So |error| <= half step of the output + w sum_j p_j |v_j| with
w = 2^-11 + 2^-12 for the tensor cores and 2^-12 for float32 arithmetic: `allowed`."""
import math

import pytest
import torch

import fp8_cache
from fp8_cache import F8, PlainCache

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def ops():
    from llm_infer_engine_b200.kernels import ops as o
    return o


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def angles(n, rot, seed=0):
    if rot == 0:
        return None
    a = torch.outer(torch.arange(n).double(), 10000.0 ** (-torch.arange(0, rot, 2).double() / rot))
    return torch.stack([torch.cos(a), torch.sin(a)], -1).float().contiguous()


def allowed(want, size, dtype, tensor_cores):
    half = torch.finfo(dtype).eps / 2
    return half * want.abs() + (2.0 ** -11 + 2.0 ** -12 if tensor_cores else 2.0 ** -12) * size + 1e-30


def same_bits(a, b):
    return torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def store(pc, qkv, table, starts, news, n_q, n_kv, hd, rot, write_kv=True, cache=None):
    """One call for sequences that bring news[i] tokens behind starts[i]; returns the rotated queries and the device cache."""
    cu = [0]
    for m in news:
        cu.append(cu[-1] + m)
    cache = pc.dev() if cache is None else cache
    q = torch.empty(cu[-1], n_q * hd, dtype=qkv.dtype, device=DEV)
    ops().rope_store_fp8(qkv.to(DEV), q, *cache, None if table is None else table.to(DEV), i32(cu), i32(pc.slots), i32(starts),
                         pc.table.to(DEV), len(news), max(news), n_q, n_kv, hd, rot, write_kv)
    return q, cache


def plain_store(pc, qkv, table, starts, news, n_q, n_kv, hd, rot):
    row, queries = 0, []
    for i, (st, m) in enumerate(zip(starts, news)):
        x = qkv[row:row + m].float().view(m, n_q + 2 * n_kv, hd)
        t = table[st:st + m] if table is not None else None
        turned = fp8_cache.rotate(x[:, :n_q + n_kv], t, rot)
        queries.append(turned[:, :n_q].reshape(m, n_q * hd).to(qkv.dtype))
        if m:
            pc.append(i, st, turned[:, n_q:], x[:, n_q + n_kv:])
        row += m
    return torch.cat(queries)


def check_cache(pc, cache, what=""):
    k, v, ke, ve = (t.cpu() for t in cache)
    assert torch.equal(ke, pc.ke) and torch.equal(ve, pc.ve), what
    assert same_bits(k, pc.k), (what, int((k.view(torch.uint8) != pc.k.view(torch.uint8)).sum()))
    assert same_bits(v, pc.v), what


# ------------------------------------------------------------------------------------------ append
LAYOUTS = [(4, 2, 16, 16), (3, 1, 32, 20), (6, 2, 48, 48), (8, 8, 64, 64), (4, 4, 64, 0), (5, 5, 80, 80), (4, 1, 96, 32),
           (16, 2, 128, 128), (20, 1, 128, 128), (2, 1, 256, 256)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("n_q,n_kv,hd,rot", LAYOUTS)
def test_append_bit_for_bit(dtype, n_q, n_kv, hd, rot):
    """Runs that begin and end inside blocks, at block and page borders, of one token and of several pages; one sequence brings
    nothing. Queries, codes and exponents are what the plain form gives; every other byte of the pages is as it was."""
    starts, news = [0, 3, 16, 70, 63, 15, 5, 128], [1, 13, 16, 9, 130, 1, 0, 33]
    pc = PlainCache([s + m for s, m in zip(starts, news)], n_kv, hd, seed=hd + n_q, nan_stale=True)
    for i, st in enumerate(starts):                    # what earlier steps left: finite
        if st:
            g = torch.Generator().manual_seed(i)
            pc.append(i, 0, torch.randn(st, n_kv, hd, generator=g), 0.1 * torch.randn(st, n_kv, hd, generator=g))
    g = torch.Generator().manual_seed(5)
    qkv = torch.randn(sum(news), (n_q + 2 * n_kv) * hd, generator=g)
    qkv *= torch.exp(2 * torch.randn(sum(news), 1, generator=g))       # some tokens raise their block's exponent, some do not
    qkv = qkv.to(dtype)
    table = angles(256, rot)
    q, cache = store(pc, qkv, table, starts, news, n_q, n_kv, hd, rot)
    want = plain_store(pc, qkv, table, starts, news, n_q, n_kv, hd, rot)
    assert torch.equal(q.cpu(), want)
    check_cache(pc, cache)
    # a step that is run again leaves what it left
    q2, cache = store(pc, qkv, table, starts, news, n_q, n_kv, hd, rot, cache=cache)
    assert torch.equal(q2, q)
    check_cache(pc, cache, "again")


@pytest.mark.parametrize("n_q,n_kv,hd", [(4, 2, 64), (4, 2, 128), (2, 1, 32)])
def test_append_holds_numbers_to_half_a_step(n_q, n_kv, hd):
    """|held - x| <= 2^-4 |x|, or half the smallest step of the block (2^-10 2^e) where x is small for its block. One call."""
    n = 77
    pc = PlainCache([n], n_kv, hd, seed=1)
    g = torch.Generator().manual_seed(2)
    qkv = (torch.randn(n, (n_q + 2 * n_kv) * hd, generator=g) * torch.exp(3 * torch.randn(n, 1, generator=g))).to(BF)
    _, cache = store(pc, qkv, angles(128, hd), [0], [n], n_q, n_kv, hd, hd)
    pc.k, pc.v, pc.ke, pc.ve = (t.cpu() for t in cache)
    x = qkv.double().view(n, n_q + 2 * n_kv, hd)
    t = angles(128, hd)[:n].double()
    a, b = x[..., :hd // 2], x[..., hd // 2:]
    c, s = t[:, None, :, 0], t[:, None, :, 1]
    turned = torch.cat([a * c - b * s, b * c + a * s], -1)[:, n_q:n_q + n_kv]
    for got, want, exps in zip(pc.held(0, n), (turned, x[:, n_q + n_kv:]), (pc.ke, pc.ve)):
        at = torch.arange(n)
        e = exps[pc.table[pc.slots[0]].long()[at // 64], :, at % 64 // 16].double()[..., None]
        # rotation in float32: three roundings of numbers up to sqrt(2) max(|a|, |b|)
        slack = 2.0 ** -22 * want.abs().amax(-1, keepdim=True) * 2
        assert bool(((got - want).abs() <= 2.0 ** -4 * want.abs() + 2.0 ** -10 * 2.0 ** e + slack).all())


@pytest.mark.parametrize("hd", [32, 64, 128])
def test_append_in_pieces(hd):
    """The same tokens one by one, in pieces and at once: the same exponents, and numbers that differ at most by the second
    rounding of codes that were small for their block (half a smallest step)."""
    n_q, n_kv, n = 2, 2, 75
    g = torch.Generator().manual_seed(3)
    qkv = (torch.randn(n, (n_q + 2 * n_kv) * hd, generator=g) * torch.exp(2 * torch.randn(n, 1, generator=g))).to(BF)
    table = angles(128, hd)
    got = []
    for cuts in ([n], [1] * n, [5, 1, 30, 12, 27]):
        pc = PlainCache([n], n_kv, hd, seed=4)
        cache, at = pc.dev(), 0
        for m in cuts:
            _, cache = store(pc, qkv[at:at + m], table, [at], [m], n_q, n_kv, hd, hd, cache=cache)
            at += m
        pc.k, pc.v, pc.ke, pc.ve = (t.cpu() for t in cache)
        got.append((pc.held(0, n), pc))
    rows = torch.arange(n)
    for (k, v), pc in got[1:]:
        pages = pc.table[pc.slots[0]].long()
        for a, b, ea, eb in ((k, got[0][0][0], pc.ke, got[0][1].ke), (v, got[0][0][1], pc.ve, got[0][1].ve)):
            ea, eb = ea[pages[rows // 64], :, rows % 64 // 16], eb[pages[rows // 64], :, rows % 64 // 16]
            assert torch.equal(ea, eb)
            assert bool(((a - b).abs() <= 2.0 ** -9 * 2.0 ** eb.double()[..., None]).all())
            assert float((a != b).double().mean()) < 0.02


@pytest.mark.parametrize("hd", [48, 64, 128])
@pytest.mark.parametrize("n_single", [1, 40, 300])
def test_append_of_a_prompt_beside_single_tokens(hd, n_single):
    """Steps in which one or two sequences bring much more than the others, some of which bring nothing, with rows behind the last."""
    n_q, n_kv = 4, 2
    g = torch.Generator().manual_seed(n_single)
    news = [1 - (i % 7 == 3) for i in range(n_single)] + [333, 0, 90]
    starts = torch.randint(0, 40, (len(news),), generator=g).tolist()
    order = torch.randperm(len(news), generator=g).tolist()
    news, starts = [news[i] for i in order], [starts[i] for i in order]
    pc = PlainCache([s + m for s, m in zip(starts, news)], n_kv, hd, seed=hd)
    for i, st in enumerate(starts):
        if st:
            pc.append(i, 0, torch.randn(st, n_kv, hd, generator=g), torch.randn(st, n_kv, hd, generator=g))
    total = sum(news)
    qkv = torch.randn(total + 5, (n_q + 2 * n_kv) * hd, generator=g).to(BF)
    table = angles(512, hd)
    cache = pc.dev()
    q = torch.full((total + 5, n_q * hd), 7.0, dtype=BF, device=DEV)
    cu = [sum(news[:i]) for i in range(len(news) + 1)]
    ops().rope_store_fp8(qkv.to(DEV), q, *cache, table.to(DEV), i32(cu), i32(pc.slots), i32(starts), pc.table.to(DEV), len(news), max(news),
                         n_q, n_kv, hd, hd)
    assert torch.equal(q[:total].cpu(), plain_store(pc, qkv[:total], table, starts, news, n_q, n_kv, hd, hd))
    assert bool((q[total:] == 7.0).all())
    check_cache(pc, cache)


@pytest.mark.parametrize("hd", [48, 64, 128])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_append_of_extreme_numbers(hd, dtype):
    """Zeros, the smallest and largest numbers of the type, and numbers that are not finite, each in a block of its own and next
    to ordinary ones; then a token that raises a block's exponent by more than its codes' range."""
    n_q, n_kv, n = 1, 1, 96
    g = torch.Generator().manual_seed(9)
    x = torch.randn(n, 3 * hd, generator=g)
    x[0:16] = 0.0
    x[16:32] = torch.finfo(dtype).tiny / 4
    x[32:48, ::3] = torch.finfo(dtype).max
    x[48:64, 5::hd] = math.inf
    x[50, 6::hd] = math.nan
    x[64:80] *= 1e-25
    x = x.to(dtype)
    pc = PlainCache([n + 8], n_kv, hd, seed=4)
    q, cache = store(pc, x, None, [0], [n], n_q, n_kv, hd, 0)
    plain_store(pc, x, None, [0], [n], n_q, n_kv, hd, 0)
    check_cache(pc, cache)
    for start, size in ((90, 1e30), (91, 1e-30)):      # as if the sequence had been cut there
        y = (torch.randn(2, 3 * hd, generator=g) * size).to(dtype)
        _, cache = store(pc, y, None, [start], [2], n_q, n_kv, hd, 0, cache=cache)
        plain_store(pc, y, None, [start], [2], n_q, n_kv, hd, 0)
        check_cache(pc, cache, size)


def test_append_without_writing_rotates_the_queries_alone():
    n_q, n_kv, hd = 4, 2, 64
    pc = PlainCache([40], n_kv, hd, seed=1)
    qkv = torch.randn(9, (n_q + 2 * n_kv) * hd).to(BF)
    before = [t.clone() for t in pc.dev()]
    q, cache = store(pc, qkv, angles(64, hd), [31], [9], n_q, n_kv, hd, hd, write_kv=False)
    for a, b in zip(before, cache):
        assert same_bits(a, b)
    want = fp8_cache.rotate(qkv.float().view(9, -1, hd)[:, :n_q], angles(64, hd)[31:40], hd)
    assert torch.equal(q.cpu(), want.reshape(9, -1).to(BF))


@pytest.mark.parametrize("hd", [32, 64])
def test_append_from_rows_that_start_anywhere(hd):
    """A step's projections that do not start on 16 bytes."""
    n_q, n_kv, n = 2, 1, 21
    pc = PlainCache([n], n_kv, hd, seed=1)
    flat = torch.randn(n * (n_q + 2 * n_kv) * hd + 1).to(BF).to(DEV)
    qkv = flat[1:].view(n, -1)
    q, cache = store(pc, qkv, angles(64, hd), [0], [n], n_q, n_kv, hd, hd)
    want = plain_store(pc, qkv.cpu(), angles(64, hd), [0], [n], n_q, n_kv, hd, hd)
    assert torch.equal(q.cpu(), want)
    check_cache(pc, cache)


# ------------------------------------------------------------------------------------------ attention
def filled(lens, n_kv, hd, seed, nan_stale=True, spread=1.0):
    """A cache whose sequences hold lens[i] positions; every other row holds what former owners left, NaN among it."""
    pc = PlainCache(lens, n_kv, hd, seed=seed, nan_stale=nan_stale)
    g = torch.Generator().manual_seed(seed)
    for i, l in enumerate(lens):
        if l:
            size = torch.exp(spread * torch.randn((l + 15) // 16, 1, 1, generator=g)).repeat_interleave(16, 0)[:l]
            pc.append(i, 0, torch.randn(l, n_kv, hd, generator=g) * size, torch.randn(l, n_kv, hd, generator=g) * size)
    return pc


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("n_q,n_kv,hd", [(4, 2, 16), (3, 1, 48), (8, 8, 64), (6, 2, 80), (4, 1, 128), (2, 1, 256)])
def test_plain_attention(dtype, n_q, n_kv, hd):
    starts, news = [0, 70, 3, 150], [33, 9, 1, 64]
    lens = [s + m for s, m in zip(starts, news)]
    pc = filled(lens, n_kv, hd, seed=hd)
    q = torch.randn(sum(news), n_q * hd, generator=torch.Generator().manual_seed(1)).to(dtype)
    tok_seq = [i for i, m in enumerate(news) for _ in range(m)]
    tok_pos = [s + j for s, m in zip(starts, news) for j in range(m)]
    for window in (0, 20, -32):
        out = torch.full((sum(news), n_q * hd), math.nan, dtype=dtype, device=DEV)
        ops().attention_paged_fp8(q.to(DEV), *pc.dev(), out, i32(tok_pos), i32(tok_seq), i32(pc.slots), pc.table.to(DEV), n_q,
                                  n_kv, hd, hd ** -0.5, window)
        row = 0
        for i, m in enumerate(news):
            k, v = pc.held(i, lens[i])
            want, size = fp8_cache.attention(q[row:row + m].double().view(m, n_q, hd), k, v, tok_pos[row:row + m], hd ** -0.5, window)
            err = (out[row:row + m].cpu().double().view(m, n_q, hd) - want).abs()
            assert bool((err <= allowed(want, size, dtype, False)).all()), (window, i, float((err / allowed(want, size, dtype, False)).max()))
            row += m


DECODE_LENS = [1, 15, 16, 17, 0, 63, 64, 65, 300, 777, 1024]


@pytest.mark.parametrize("window", [0, 40, 1000, -64])
@pytest.mark.parametrize("n_q,n_kv,hd", [(4, 4, 64), (12, 4, 64), (8, 1, 64), (13, 1, 64), (32, 8, 128), (40, 8, 128), (16, 1, 128),
                                         (20, 1, 128), (20, 1, 64)])
def test_decode(n_q, n_kv, hd, window):
    """Lengths around blocks and pages, a sequence that holds nothing, groups of 1 to 20 query heads."""
    pc = filled(DECODE_LENS, n_kv, hd, seed=hd + n_q)
    n = len(DECODE_LENS)
    q = torch.randn(n, n_q * hd, generator=torch.Generator().manual_seed(1)).to(BF)
    out = torch.full((n, n_q * hd), math.nan, dtype=BF, device=DEV)
    ops().attention_decode_fp8(q.to(DEV), *pc.dev(), out, i32(pc.slots), i32(DECODE_LENS), pc.table.to(DEV), n_q, n_kv, hd,
                               hd ** -0.5, window, 1024)
    for i, l in enumerate(DECODE_LENS):
        if l == 0:
            assert bool((out[i] == 0).all())
            continue
        want, size = fp8_cache.attention(q[i:i + 1].double().view(1, n_q, hd), *pc.held(i, l), [l - 1], hd ** -0.5, window)
        err = (out[i].cpu().double().view(1, n_q, hd) - want).abs()
        assert bool((err <= allowed(want, size, BF, True)).all()), (l, float((err / allowed(want, size, BF, True)).max()))


@pytest.mark.parametrize("n,n_q,n_kv,hd", [(18, 32, 8, 64), (20, 14, 2, 64), (18, 40, 4, 64), (37, 28, 4, 128), (18, 48, 4, 128),
                                           (18, 32, 8, 128), (40, 32, 8, 128), (80, 32, 8, 64)])
@pytest.mark.parametrize("longest", [70, 1100])
def test_decode_of_some_dozen_sequences(n, n_q, n_kv, hd, longest):
    """Between a few items, which have several blocks each, and many, which share blocks: large blocks, alone or in pairs. With the
    longest length named and not; a step on top of it leaves what appending and attending leaves."""
    g = torch.Generator().manual_seed(n + hd)
    lens = torch.randint(1, longest, (n,), generator=g).tolist()
    lens[3], lens[5] = longest, 0
    pc = filled(lens, n_kv, hd, seed=n)
    q = torch.randn(n, n_q * hd, generator=g).to(BF)
    outs = []
    for max_len in (longest, 0):
        out = torch.full((n, n_q * hd), math.nan, dtype=BF, device=DEV)
        ops().attention_decode_fp8(q.to(DEV), *pc.dev(), out, i32(pc.slots), i32(lens), pc.table.to(DEV), n_q, n_kv, hd, hd ** -0.5, 0,
                                   max_len)
        outs.append(out)
        for i, l in enumerate(lens):
            if l == 0:
                assert bool((out[i] == 0).all())
                continue
            want, size = fp8_cache.attention(q[i:i + 1].double().view(1, n_q, hd), *pc.held(i, l), [l - 1], hd ** -0.5, 0)
            err = (out[i].cpu().double().view(1, n_q, hd) - want).abs()
            assert bool((err <= allowed(want, size, BF, True)).all()), (i, l, float((err / allowed(want, size, BF, True)).max()))
    # the step of the last tokens, whose keys and values are in place already: an append of the same numbers
    starts, news = [max(l - 1, 0) for l in lens], [min(l, 1) for l in lens]
    qkv = torch.randn(n, (n_q + 2 * n_kv) * hd, generator=g).to(BF)
    table = angles(longest, hd)
    rows = torch.tensor([i for i, m in enumerate(news) if m])
    rotated, after = store(pc, qkv[rows], table, starts, news, n_q, n_kv, hd, hd)
    for max_len in (longest, 0):
        stepped, out = pc.dev(), torch.zeros(n, n_q * hd, dtype=BF, device=DEV)
        ops().attention_decode_fp8_rope(qkv.to(DEV), *stepped, out, table.to(DEV), i32(pc.slots), i32(lens), pc.table.to(DEV), n_q, n_kv,
                                        hd, hd ** -0.5, 0, max_len)
        assert all(same_bits(a, b) for a, b in zip(stepped, after))
        whole = torch.zeros(n, n_q * hd, dtype=BF, device=DEV)
        x = torch.zeros(n, n_q * hd, dtype=BF, device=DEV)
        x[rows.to(DEV)] = rotated
        ops().attention_decode_fp8(x, *after, whole, i32(pc.slots), i32(lens), pc.table.to(DEV), n_q, n_kv, hd, hd ** -0.5, 0, max_len)
        assert torch.equal(out, whole)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("case", ["large keys", "small queries", "large queries", "values apart", "zero values", "negative scale"])
def test_decode_far_ranges(hd, case):
    """Scores, queries and values far from 1: the sum over the values is in half precision inside, the ranges are not."""
    n_q, n_kv, lens = 8, 2, [200, 333]
    g = torch.Generator().manual_seed(3)
    pc = PlainCache(lens, n_kv, hd, seed=5)
    q = torch.randn(2, n_q * hd, generator=g)
    scale = hd ** -0.5
    k_size = v_size = None
    if case == "large keys":
        k_size, scale = 1e18, 1e-18 * hd ** -0.5
    elif case == "small queries":
        q, scale = q * 1e-20, 1e20 * hd ** -0.5
    elif case == "large queries":
        q, scale = q * 1e20, 1e-20 * hd ** -0.5
    elif case == "negative scale":
        scale = -scale
    for i, l in enumerate(lens):
        k, v = torch.randn(l, n_kv, hd, generator=g), torch.randn(l, n_kv, hd, generator=g)
        if k_size:
            k = k * k_size
        if case == "values apart":                     # blocks of values from 1e-12 to 1e12
            v = v * (10.0 ** torch.linspace(-12, 12, (l + 15) // 16).repeat_interleave(16)[:l, None, None])
        if case == "zero values":
            v[16:l - 20] = 0.0
        pc.append(i, 0, k, v)
    q = q.to(BF)
    out = torch.empty(2, n_q * hd, dtype=BF, device=DEV)
    ops().attention_decode_fp8(q.to(DEV), *pc.dev(), out, i32(pc.slots), i32(lens), pc.table.to(DEV), n_q, n_kv, hd, scale, 0, 333)
    for i, l in enumerate(lens):
        want, size = fp8_cache.attention(q[i:i + 1].double().view(1, n_q, hd), *pc.held(i, l), [l - 1], scale, 0)
        err = (out[i].cpu().double().view(1, n_q, hd) - want).abs()
        assert bool((err <= allowed(want, size, BF, True)).all()), float((err / allowed(want, size, BF, True)).max())


def test_decode_numbers_that_are_not_finite_stay_with_the_rows_that_see_them():
    """A key or value that is NaN, a query head that is: NaN where they are seen, nothing elsewhere."""
    n_q, n_kv, hd, lens = 8, 2, 64, [100, 100, 100, 100]
    pc = filled(lens, n_kv, hd, seed=8)
    g = torch.Generator().manual_seed(8)
    k, v = torch.randn(1, n_kv, hd, generator=g), torch.randn(1, n_kv, hd, generator=g)
    bad_k, bad_v = k.clone(), v.clone()
    bad_k[0, 1, 3], bad_v[0, 1, 5] = math.inf, math.nan
    pc.append(0, 50, bad_k, v)                         # sequence 0: a key of KV head 1 is not finite
    pc.append(1, 50, k, bad_v)                         # sequence 1: one column of a value of KV head 1
    q = torch.randn(4, n_q * hd, generator=g).to(BF)
    q[2, 3 * hd + 1] = math.inf                        # sequence 2: query head 3
    out = torch.empty(4, n_q * hd, dtype=BF, device=DEV)
    for window, seen in ((0, True), (40, False)):
        ops().attention_decode_fp8(q.to(DEV), *pc.dev(), out, i32(pc.slots), i32(lens), pc.table.to(DEV), n_q, n_kv, hd, 0.125,
                                   window, 100)
        bad = torch.isnan(out.cpu()).view(4, n_q, hd)
        want = torch.zeros_like(bad)
        if seen:
            want[0, 4:] = True
            want[1, 4:, 5] = True
        want[2, 3] = True
        assert torch.equal(bad, want), window


def test_decode_of_one_long_sequence_among_short_ones():
    """A sequence that is cut into many shares, beside ones of a block: a needle far back must come through."""
    n_q, n_kv, hd = 8, 2, 128
    lens = [5, 20000, 1, 40]
    pc = filled(lens, n_kv, hd, seed=2, spread=0.3)
    q = torch.randn(4, n_q * hd, generator=torch.Generator().manual_seed(2)).to(BF)
    needle = q[1].float().view(n_q, hd)[::n_q // n_kv]
    needle = needle * (24.0 / ((needle * needle).sum(-1, keepdim=True) * hd ** -0.5))
    pc.append(1, 1234, needle[None], torch.full((1, n_kv, hd), 5.0))
    out = torch.empty(4, n_q * hd, dtype=BF, device=DEV)
    for max_len in (20000, 0):
        ops().attention_decode_fp8(q.to(DEV), *pc.dev(), out, i32(pc.slots), i32(lens), pc.table.to(DEV), n_q, n_kv, hd,
                                   hd ** -0.5, 0, max_len)
        for i, l in enumerate(lens):
            want, size = fp8_cache.attention(q[i:i + 1].double().view(1, n_q, hd), *pc.held(i, l), [l - 1], hd ** -0.5, 0)
            err = (out[i].cpu().double().view(1, n_q, hd) - want).abs()
            # 20,000 keys: eight times the keys that `allowed` counts float32 sums for
            assert bool((err <= allowed(want, size, BF, True) + 2.0 ** -10 * size).all()), l
        assert float(out[1].float().view(n_q, hd)[::n_q // n_kv].mean()) > 4.0


# ------------------------------------------------------------------------------------------ prompts
def prompt(pc, q, starts, news, n_q, n_kv, hd, scale, window, cache=None):
    cu = [0]
    for m in news:
        cu.append(cu[-1] + m)
    out = torch.full((cu[-1], n_q * hd), math.nan, dtype=BF, device=DEV)
    ops().attention_prefill_fp8(q.to(DEV), *(pc.dev() if cache is None else cache), out, i32(cu), i32(pc.slots), i32(starts),
                                pc.table.to(DEV), len(news), max(news), n_q, n_kv, hd, scale, window)
    ops().check_tc_status(DEV)
    return out.cpu().double()


def check_prompt(pc, out, q, starts, news, n_q, n_kv, hd, scale, window, rows=None):
    """Every row, or `rows` of each sequence's."""
    row = 0
    for i, (st, m) in enumerate(zip(starts, news)):
        pick = list(range(m)) if rows is None else sorted({r for r in rows if r < m} | ({m - 1} if m else set()))
        if pick:
            want, size = fp8_cache.attention(q[row:row + m].double().view(m, n_q, hd)[pick], *pc.held(i, st + m),
                                             [st + r for r in pick], scale, window)
            err = (out[row:row + m].view(m, n_q, hd)[pick] - want).abs()
            bound = allowed(want, size, BF, True)
            assert bool((err <= bound).all()), (i, st, m, float((err / bound).max()), int((err > bound).sum()))
        row += m


@pytest.mark.parametrize("n_q,n_kv,hd", [(4, 1, 64), (4, 1, 128)])
@pytest.mark.parametrize("start,new", [(0, 2), (0, 33), (100, 28)])
def test_prompt_small(n_q, n_kv, hd, start, new):
    pc = filled([start + new], n_kv, hd, seed=hd)
    q = torch.randn(new, n_q * hd, generator=torch.Generator().manual_seed(1)).to(BF)
    out = prompt(pc, q, [start], [new], n_q, n_kv, hd, hd ** -0.5, 0)
    check_prompt(pc, out, q, [start], [new], n_q, n_kv, hd, hd ** -0.5, 0)


@pytest.mark.parametrize("window", [0, 40, 200, -64, -300])
@pytest.mark.parametrize("n_q,n_kv,hd", [(2, 2, 64), (12, 4, 64), (7, 1, 128), (8, 2, 128), (16, 1, 64), (40, 1, 64)])
def test_prompt(n_q, n_kv, hd, window):
    """Ragged pieces at odd places, one of a token, one of none; groups of 1 to 40 query heads."""
    starts, news = [0, 70, 3, 700, 130, 63], [33, 9, 1, 40, 300, 0]
    pc = filled([s + m for s, m in zip(starts, news)], n_kv, hd, seed=hd + n_q)
    q = torch.randn(sum(news), n_q * hd, generator=torch.Generator().manual_seed(1)).to(BF)
    out = prompt(pc, q, starts, news, n_q, n_kv, hd, hd ** -0.5, window)
    check_prompt(pc, out, q, starts, news, n_q, n_kv, hd, hd ** -0.5, window, rows=[0, 1, 15, 16, 31, 32, 63, 64, 127, 128, 129, 255])


@pytest.mark.parametrize("n_q,n_kv,hd,start,new", [(4, 1, 64, 0, 1500), (8, 2, 128, 400, 1100), (4, 4, 64, 0, 700), (8, 1, 128, 3000, 5)])
def test_prompt_long(n_q, n_kv, hd, start, new):
    """Many key tiles: the bound moves, the sums are rescaled, tiles are cut into runs and joined. A needle early on."""
    pc = filled([start + new], n_kv, hd, seed=3, spread=0.5)
    g = torch.Generator().manual_seed(4)
    q = torch.randn(new, n_q * hd, generator=g).to(BF)
    needle = q[-1].float().view(n_q, hd)[::n_q // n_kv]
    needle = needle * (24.0 / ((needle * needle).sum(-1, keepdim=True) * hd ** -0.5))
    pc.append(0, 7, needle[None], torch.full((1, n_kv, hd), 5.0))
    out = prompt(pc, q, [start], [new], n_q, n_kv, hd, hd ** -0.5, 0)
    check_prompt(pc, out, q, [start], [new], n_q, n_kv, hd, hd ** -0.5, 0, rows=[0, 1, 100, 127, 128, 511, 512, 640, 1000])
    assert float(out[-1].view(n_q, hd)[::n_q // n_kv].mean()) > 4.0


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("case", ["large keys", "small queries", "large queries", "values apart", "zero values", "zero queries",
                                  "growing scores"])
def test_prompt_far_ranges(hd, case):
    n_q, n_kv, starts, news = 4, 2, [150, 0], [40, 300]
    g = torch.Generator().manual_seed(3)
    pc = PlainCache([s + m for s, m in zip(starts, news)], n_kv, hd, seed=5, nan_stale=True)
    q = torch.randn(sum(news), n_q * hd, generator=g)
    scale = hd ** -0.5
    for i, l in enumerate(s + m for s, m in zip(starts, news)):
        k, v = torch.randn(l, n_kv, hd, generator=g), torch.randn(l, n_kv, hd, generator=g)
        if case == "large keys":
            k = k * 1e18
        if case == "values apart":
            v = v * (10.0 ** torch.linspace(-12, 12, (l + 15) // 16).repeat_interleave(16)[:l, None, None])
        if case == "zero values":
            v[16:l - 20] = 0.0
        if case == "zero queries":
            k[:64] = 0.0
        if case == "growing scores":                   # every key tile has larger scores than the one before
            k = k * torch.linspace(0.1, 12.0, l)[:, None, None]
        pc.append(i, 0, k, v)
    if case == "large keys":
        scale *= 1e-18
    elif case == "small queries":
        q, scale = q * 1e-20, scale * 1e20
    elif case == "large queries":
        q, scale = q * 1e20, scale * 1e-20
    elif case == "zero queries":
        q[:] = 0.0
    q = q.to(BF)
    out = prompt(pc, q, starts, news, n_q, n_kv, hd, scale, 0)
    check_prompt(pc, out, q, starts, news, n_q, n_kv, hd, scale, 0, rows=[0, 1, 17, 100, 128, 200])


@pytest.mark.parametrize("hd", [64, 128])
def test_prompt_numbers_that_are_not_finite_stay_with_the_rows_that_see_them(hd):
    n_q, n_kv, new = 4, 2, 200
    pc = filled([new], n_kv, hd, seed=8)
    g = torch.Generator().manual_seed(8)
    k, v = torch.randn(1, n_kv, hd, generator=g), torch.randn(1, n_kv, hd, generator=g)
    bad_k, bad_v = k.clone(), v.clone()
    bad_k[0, 1, 3], bad_v[0, 0, 5] = math.inf, math.nan
    pc.append(0, 60, k, bad_v)                         # position 60: column 5 of KV head 0's value
    pc.append(0, 130, bad_k, v)                        # position 130: the key of KV head 1
    q = torch.randn(new, n_q * hd, generator=g).to(BF)
    q[20, 3 * hd + 1] = math.nan                       # one query head of one token
    for window in (0, 30):
        bad = torch.isnan(prompt(pc, q, [0], [new], n_q, n_kv, hd, hd ** -0.5, window)).view(new, n_q, hd)
        want = torch.zeros_like(bad)
        last = new if window == 0 else None
        want[60:last or 90, :2, 5] = True
        want[130:last or 160, 2:] = True
        want[20, 3] = True
        assert torch.equal(bad, want), window


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n_kv,n_short,longs", [(1, 147, [2000]), (1, 130, [2000, 1900]), (1, 128, [2500]), (2, 90, [2000]),
                                                (1, 20, [2500, 600, 1300]), (4, 30, [2000, 1000, 900])])
def test_prompt_cut_beside_short_ones(hd, n_kv, n_short, longs):
    """Some sequences are cut into runs and others are not, with fewer tiles of tokens than SMs, as many, and more."""
    n_q = 4 * n_kv
    starts, news = [0] * n_short + longs, [1 + i % 3 for i in range(n_short)] + [5] * len(longs)
    order = torch.randperm(len(news), generator=torch.Generator().manual_seed(7)).tolist()
    starts, news = [starts[i] for i in order], [news[i] for i in order]
    pc = filled([s + m for s, m in zip(starts, news)], n_kv, hd, seed=n_short)
    q = torch.randn(sum(news), n_q * hd, generator=torch.Generator().manual_seed(1)).to(BF)
    out = prompt(pc, q, starts, news, n_q, n_kv, hd, hd ** -0.5, 0)
    check_prompt(pc, out, q, starts, news, n_q, n_kv, hd, hd ** -0.5, 0)


@pytest.mark.parametrize("hd", [64, 128])
def test_prompt_of_few_tokens_in_a_large_step(hd):
    """More rows than the sequences have: those behind the last one stay as they were, and how the others' work is cut, which is
    found by the lengths that are there, has room for its runs whatever the rows made the caller count on."""
    n_q, n_kv, starts, news = 8, 2, [2500, 0, 700], [3, 40, 200]
    pc = filled([s + m for s, m in zip(starts, news)], n_kv, hd, seed=5)
    rows = 40000
    q = torch.randn(rows, n_q * hd, generator=torch.Generator().manual_seed(1)).to(BF)
    cu = i32([0, 3, 43, 243])
    for most in (200, 4000):
        out = torch.full((rows, n_q * hd), 3.0, dtype=BF, device=DEV)
        ops().attention_prefill_fp8(q.to(DEV), *pc.dev(), out, cu, i32(pc.slots), i32(starts), pc.table.to(DEV), 3, most, n_q, n_kv, hd,
                                    hd ** -0.5, 0)
        ops().check_tc_status(DEV)
        assert bool((out[243:] == 3.0).all())
        check_prompt(pc, out[:243].cpu().double(), q, starts, news, n_q, n_kv, hd, hd ** -0.5, 0, rows=[0, 1, 2, 39, 63, 64, 128])


@pytest.mark.parametrize("hd", [64, 128])
def test_prompt_nan_in_one_run_of_several(hd):
    """A value that is not finite reaches its column of the rows that see it, through the join; a key its rows."""
    n_q, n_kv, start, new = 4, 1, 2500, 6
    pc = filled([start + new, start + new], n_kv, hd, seed=9)
    v = torch.randn(1, n_kv, hd, generator=torch.Generator().manual_seed(2))
    v[0, 0, 5] = math.inf
    pc.append(0, 300, torch.zeros(1, n_kv, hd), v)
    v[0, 0, 5], v[0, 0, hd - 1] = 1.0, math.nan
    pc.append(0, start + 3, torch.zeros(1, n_kv, hd), v)
    pc.append(1, start + 2, torch.full((1, n_kv, hd), math.nan), torch.ones(1, n_kv, hd))
    q = torch.randn(2 * new, n_q * hd, generator=torch.Generator().manual_seed(1)).to(BF)
    bad = torch.isnan(prompt(pc, q, [start, start], [new, new], n_q, n_kv, hd, hd ** -0.5, 0)).view(2, new, n_q, hd)
    want = torch.zeros(2, new, n_q, hd, dtype=torch.bool)
    want[0, :, :, 5] = True
    want[0, 3:, :, hd - 1] = True
    want[1, 2:] = True
    assert torch.equal(bad, want)


# ------------------------------------------------------------------------------------------ one-token steps in one kernel
@pytest.mark.parametrize("window", [0, 40, -64])
@pytest.mark.parametrize("n_q,n_kv,hd", [(4, 4, 64), (12, 4, 64), (32, 8, 128), (7, 1, 128), (16, 1, 64), (32, 2, 128)])
def test_step(n_q, n_kv, hd, window):
    """The new key and value go into the cache bit for bit as rope_store_fp8 leaves them (blocks that begin, go on, raise their
    exponent), and attention sees them; a lane without a sequence writes nothing. Run twice: the same."""
    lens = [1, 16, 17, 64, 65, 300, 0, 777, 48]
    n = len(lens)
    pc = PlainCache(lens, n_kv, hd, seed=hd + n_q, nan_stale=True)
    g = torch.Generator().manual_seed(3)
    for i, l in enumerate(lens):
        if l > 1:
            pc.append(i, 0, torch.randn(l - 1, n_kv, hd, generator=g), torch.randn(l - 1, n_kv, hd, generator=g))
    qkv = torch.randn(n, (n_q + 2 * n_kv) * hd, generator=g)
    qkv[2] *= 40.0                                     # position 16 begins a block
    qkv[5] *= 40.0                                     # position 299 raises its block's exponents
    qkv[8] *= 1e-3                                     # position 47 does not
    qkv = qkv.to(BF)
    table = angles(1024, hd)
    cache = pc.dev()
    before = [t.clone() for t in cache]
    outs = []
    for _ in range(2):
        out = torch.full((n, n_q * hd), math.nan, dtype=BF, device=DEV)
        ops().attention_decode_fp8_rope(qkv.to(DEV), *cache, out, table.to(DEV), i32(pc.slots), i32(lens), pc.table.to(DEV), n_q,
                                        n_kv, hd, hd ** -0.5, window, 1024)
        outs.append(out)
    assert torch.equal(outs[0], outs[1])
    starts, news = [max(l - 1, 0) for l in lens], [min(l, 1) for l in lens]
    keep = torch.tensor([m > 0 for m in news])
    q = plain_store(pc, qkv[keep], table, starts, news, n_q, n_kv, hd, hd)
    check_cache(pc, cache)
    assert not same_bits(before[0], cache[0])
    row = 0
    for i, l in enumerate(lens):
        if l == 0:
            assert bool((outs[0][i] == 0).all())
            continue
        want, size = fp8_cache.attention(q[row:row + 1].double().view(1, n_q, hd), *pc.held(i, l), [l - 1], hd ** -0.5, window)
        err = (outs[0][i].cpu().double().view(1, n_q, hd) - want).abs()
        assert bool((err <= allowed(want, size, BF, True)).all()), (l, float((err / allowed(want, size, BF, True)).max()))
        row += 1


# ------------------------------------------------------------------------------------------ calls at the edges
class FarPages:
    """A plain cache's pages at the end of a device cache of `pages` pages, whose other pages nobody looks at."""

    def __init__(self, pc, pages):
        self.pc, self.first = pc, pages - pc.n_pages
        shape = (pages, pc.n_kv, 64, pc.hd)
        self.cache = [torch.empty(shape, dtype=F8, device=DEV), torch.empty(shape, dtype=F8, device=DEV),
                      torch.empty(shape[:2] + (4,), dtype=torch.int8, device=DEV), torch.empty(shape[:2] + (4,), dtype=torch.int8, device=DEV)]
        for far, near in zip(self.cache, pc.dev()):
            far.view(torch.uint8)[self.first:] = near.view(torch.uint8)
        self.table = (pc.table + self.first).to(DEV)

    def back(self):
        return [t[self.first:] for t in self.cache]


def test_pages_behind_the_first_four_billion_codes():
    """Offsets of codes pass 32 bits: every call on pages at the end of caches of 4.6 GB each."""
    n_q, n_kv, hd = 16, 8, 128
    lens, new = [130, 77], [33, 9]
    pc = PlainCache(lens, n_kv, hd, seed=11)
    g = torch.Generator().manual_seed(12)
    starts = [l - m for l, m in zip(lens, new)]
    for i, st in enumerate(starts):
        pc.append(i, 0, torch.randn(st, n_kv, hd, generator=g), torch.randn(st, n_kv, hd, generator=g))
    far = FarPages(pc, 70000)
    assert far.first * n_kv * 64 * hd > 2 ** 32
    qkv = torch.randn(sum(new), (n_q + 2 * n_kv) * hd, generator=g).to(BF)
    table = angles(256, hd)
    q = torch.empty(sum(new), n_q * hd, dtype=BF, device=DEV)
    cu = i32([0, new[0], sum(new)])
    ops().rope_store_fp8(qkv.to(DEV), q, *far.cache, table.to(DEV), cu, i32(pc.slots), i32(starts), far.table, 2, max(new), n_q, n_kv,
                         hd, hd)
    assert torch.equal(q.cpu(), plain_store(pc, qkv, table, starts, new, n_q, n_kv, hd, hd))
    check_cache(pc, far.back())
    out = torch.empty_like(q)
    ops().attention_prefill_fp8(q, *far.cache, out, cu, i32(pc.slots), i32(starts), far.table, 2, max(new), n_q, n_kv, hd, hd ** -0.5)
    check_prompt(pc, out.cpu().double(), q.cpu(), starts, new, n_q, n_kv, hd, hd ** -0.5, 0)
    plain = torch.empty_like(q)
    pos = [st + j for st, m in zip(starts, new) for j in range(m)]
    ops().attention_paged_fp8(q, *far.cache, plain, i32(pos), i32([0] * new[0] + [1] * new[1]), i32(pc.slots), far.table, n_q, n_kv, hd,
                              hd ** -0.5)
    check_prompt(pc, plain.cpu().double(), q.cpu(), starts, new, n_q, n_kv, hd, hd ** -0.5, 0)
    last = q[[new[0] - 1, sum(new) - 1]].contiguous()
    for max_len in (130, 0):
        got = torch.empty_like(last)
        ops().attention_decode_fp8(last, *far.cache, got, i32(pc.slots), i32(lens), far.table, n_q, n_kv, hd, hd ** -0.5, 0, max_len)
        row = 0
        for i, l in enumerate(lens):
            want, size = fp8_cache.attention(last[i:i + 1].cpu().double().view(1, n_q, hd), *pc.held(i, l), [l - 1], hd ** -0.5, 0)
            assert bool(((got[i].cpu().double().view(1, n_q, hd) - want).abs() <= allowed(want, size, BF, True)).all())
    step = torch.randn(2, (n_q + 2 * n_kv) * hd, generator=g).to(BF)
    got = torch.empty_like(last)
    ops().attention_decode_fp8_rope(step.to(DEV), *far.cache, got, table.to(DEV), i32(pc.slots), i32(lens), far.table, n_q, n_kv, hd,
                                    hd ** -0.5)
    plain_store(pc, step, table, [l - 1 for l in lens], [1, 1], n_q, n_kv, hd, hd)
    check_cache(pc, far.back())


@pytest.mark.parametrize("hd", [64, 128])
def test_captured_calls_follow_the_lengths_that_are_there(hd):
    """A step, a prompt and their joins captured once and replayed with other lengths, tables and tokens: what eager calls give."""
    n_q, n_kv, n = 8, 2, 6
    table = angles(4096, hd).to(DEV)
    longest = [2000, 40, 700, 64, 1, 300]
    pc = filled(longest, n_kv, hd, seed=4)
    cache = [t.clone() for t in pc.dev()]
    fresh = [t.clone() for t in cache]
    slots, lens, pages = i32(pc.slots), i32([1] * n), pc.table.to(DEV)
    starts, cu = i32([0] * n), i32([0, 1, 2, 3, 4, 5, 6])
    qkv = torch.zeros(n, (n_q + 2 * n_kv) * hd, dtype=BF, device=DEV)
    q = torch.zeros(64, n_q * hd, dtype=BF, device=DEV)
    outs = [torch.zeros(n, n_q * hd, dtype=BF, device=DEV), torch.zeros(n, n_q * hd, dtype=BF, device=DEV), torch.zeros_like(q)]

    def calls():
        ops().attention_decode_fp8_rope(qkv, *cache, outs[0], table, slots, lens, pages, n_q, n_kv, hd, hd ** -0.5)
        ops().attention_decode_fp8(q[:n], *cache, outs[1], slots, lens, pages, n_q, n_kv, hd, hd ** -0.5, 0, 64)
        ops().attention_prefill_fp8(q, *cache, outs[2], cu, slots, starts, pages, n, 64, n_q, n_kv, hd, hd ** -0.5)

    calls()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls()
    g = torch.Generator().manual_seed(5)
    for held, news in (([2000, 40, 700, 64, 1, 300], [3, 9, 1, 20, 1, 30]), ([5, 1, 0, 33, 1, 0], [1, 1, 0, 33, 1, 0]),
                       ([1999, 39, 0, 0, 0, 0], [64, 0, 0, 0, 0, 0]), ([0] * 6, [0] * 6)):
        results = []
        for run in (graph.replay, calls):
            for t, f in zip(cache, fresh):
                t.copy_(f)
            lens.copy_(torch.tensor(held))
            starts.copy_(torch.tensor([max(h - m, 0) for h, m in zip(held, news)]))
            cu.copy_(torch.tensor([sum(news[:i]) for i in range(n + 1)]))
            g.manual_seed(6)
            qkv.copy_(torch.randn(qkv.shape, generator=g))
            q.copy_(torch.randn(q.shape, generator=g))
            for o in outs:
                o.fill_(7.0)
            run()
            torch.cuda.synchronize()
            ops().check_tc_status(DEV)
            results.append([o.clone() for o in outs] + [t.clone() for t in cache])
        assert all(same_bits(a, b) for a, b in zip(*results))
        assert bool((results[0][2][sum(news):] == 7.0).all())
        for i, h in enumerate(held):
            if h == 0:
                assert bool((results[0][0][i] == 0).all()) and bool((results[0][1][i] == 0).all())


@pytest.mark.parametrize("hd", [64, 128])
def test_two_streams_at_once(hd):
    """Calls that need scratch, on two streams and as two captured graphs at once, leave what one call leaves."""
    n_q, n_kv = 8, 2
    lens = [6000, 900, 3500, 20, 1, 2000, 700, 64]
    pc = filled(lens, n_kv, hd, seed=3)
    cache, slots, held, pages = pc.dev(), i32(pc.slots), i32(lens), pc.table.to(DEV)
    n = len(lens)
    starts, cu = i32([l - 1 for l in lens]), i32(list(range(n + 1)))
    qs = [torch.randn(n, n_q * hd, generator=torch.Generator().manual_seed(s)).to(BF).to(DEV) for s in (1, 2)]

    def calls(q):
        a, b = torch.empty_like(q), torch.empty_like(q)
        ops().attention_decode_fp8(q, *cache, a, slots, held, pages, n_q, n_kv, hd, hd ** -0.5)
        ops().attention_prefill_fp8(q, *cache, b, cu, slots, starts, pages, n, 1, n_q, n_kv, hd, hd ** -0.5)
        return a, b

    want = [calls(q) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    graphs, graph_outs = [], []
    for q in qs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            graph_outs.append(calls(q))
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(calls(qs[i]))
                graphs[i].replay()
    torch.cuda.synchronize()
    ops().check_tc_status(DEV)
    for i in range(2):
        for pair in got[i] + [graph_outs[i]]:
            assert torch.equal(pair[0], want[i][0]) and torch.equal(pair[1], want[i][1])


def test_more_tokens_than_the_table_has_room_for():
    """Lengths beyond the table (a caller's mistake): nothing is written or read outside the sequence's pages."""
    n_q, n_kv, hd = 8, 2, 64
    pc = filled([128, 128], n_kv, hd, seed=2)
    table = pc.table[:, :2].contiguous()               # two pages a sequence
    cache = pc.dev()
    before = [t.clone() for t in cache]
    qkv = torch.randn(2, (n_q + 2 * n_kv) * hd, generator=torch.Generator().manual_seed(1)).to(BF).to(DEV)
    angle = angles(64, hd).to(DEV)                     # and fewer angles than positions
    out = torch.empty(2, n_q * hd, dtype=BF, device=DEV)
    ops().attention_decode_fp8_rope(qkv, *cache, out, angle, i32(pc.slots), i32([129, 1000]), table.to(DEV), n_q, n_kv, hd, hd ** -0.5)
    assert all(same_bits(a, b) for a, b in zip(before, cache))
    q = torch.zeros(2, n_q * hd, dtype=BF, device=DEV)
    ops().rope_store_fp8(qkv, q, *cache, angle, i32([0, 1, 2]), i32(pc.slots), i32([128, 999]), table.to(DEV), 2, 1, n_q, n_kv, hd, hd)
    assert all(same_bits(a, b) for a, b in zip(before, cache))
    x = torch.randn(2, n_q * hd, generator=torch.Generator().manual_seed(3)).to(BF)
    want = torch.cat([fp8_cache.attention(x[i:i + 1].double().view(1, n_q, hd), *pc.held(i, 128), [127], hd ** -0.5, 0)[0] for i in range(2)])
    for call in ("decode", "prefill", "plain"):
        out.fill_(math.nan)
        if call == "decode":
            ops().attention_decode_fp8(x.to(DEV), *cache, out, i32(pc.slots), i32([129, 1000]), table.to(DEV), n_q, n_kv, hd, hd ** -0.5)
        elif call == "prefill":
            ops().attention_prefill_fp8(x.to(DEV), *cache, out, i32([0, 1, 2]), i32(pc.slots), i32([128, 999]), table.to(DEV), 2, 1, n_q,
                                        n_kv, hd, hd ** -0.5)
        else:
            ops().attention_paged_fp8(x.to(DEV), *cache, out, i32([128, 999]), i32([0, 1]), i32(pc.slots), table.to(DEV), n_q, n_kv, hd,
                                      hd ** -0.5)
        err = (out[0].cpu().double().view(n_q, hd) - want[0]).abs()
        assert float(err.max()) < 0.1, call            # every key that there is, where the call can tell


def test_calls_with_nothing_to_do():
    n_q, n_kv, hd = 4, 2, 64
    pc = PlainCache([10], n_kv, hd)
    cache, none = pc.dev(), torch.empty(0, n_q * hd, dtype=BF, device=DEV)
    before = [t.clone() for t in cache]
    empty = torch.empty(0, dtype=torch.int32, device=DEV)
    pages = pc.table.to(DEV)
    ops().rope_store_fp8(torch.empty(0, (n_q + 2 * n_kv) * hd, dtype=BF, device=DEV), none, *cache, None, i32([0]), empty, empty, pages, 0, 0,
                         n_q, n_kv, hd, 0)
    ops().attention_paged_fp8(none, *cache, none, empty, empty, empty, pages, n_q, n_kv, hd, 0.1)
    ops().attention_decode_fp8(none, *cache, none, empty, empty, pages, n_q, n_kv, hd, 0.1)
    ops().attention_decode_fp8_rope(torch.empty(0, (n_q + 2 * n_kv) * hd, dtype=BF, device=DEV), *cache, none, angles(8, hd).to(DEV), empty,
                                    empty, pages, n_q, n_kv, hd, 0.1)
    ops().attention_prefill_fp8(none, *cache, none, i32([0]), empty, empty, pages, 0, 0, n_q, n_kv, hd, 0.1)
    torch.cuda.synchronize()
    assert all(same_bits(a, b) for a, b in zip(before, cache))


def good_call(name):
    """Arguments of a call that is taken, by name."""
    n_q, n_kv, hd, n = 4, 2, 64, 2
    pc = filled([20, 30], n_kv, hd, seed=1)
    k, v, ke, ve = pc.dev()
    a = dict(k_cache=k, v_cache=v, k_exp=ke, v_exp=ve, seq_slot=i32(pc.slots), block_table=pc.table.to(DEV), n_q=n_q, n_kv=n_kv,
             head_dim=hd)
    q, qkv = torch.zeros(n, n_q * hd, dtype=BF, device=DEV), torch.zeros(n, (n_q + 2 * n_kv) * hd, dtype=BF, device=DEV)
    packed = dict(cu_q=i32([0, 1, 2]), seq_start=i32([19, 29]), n_seqs=2, max_q_len=1)
    if name == "rope_store_fp8":
        return dict(a, qkv=qkv, q_out=q, table=angles(64, hd).to(DEV), rot_dim=hd, **packed)
    if name == "attention_paged_fp8":
        return dict(a, q=q, out=torch.zeros_like(q), tok_pos=i32([19, 29]), tok_seq=i32([0, 1]), scale=0.1)
    if name == "attention_decode_fp8":
        return dict(a, q=q, out=torch.zeros_like(q), seq_kvlen=i32([20, 30]), scale=0.1)
    if name == "attention_decode_fp8_rope":
        return dict(a, qkv=qkv, out=q, table=angles(64, hd).to(DEV), seq_kvlen=i32([20, 30]), scale=0.1)
    return dict(a, q=q, out=torch.zeros_like(q), scale=0.1, **packed)


def shifted(t):
    """The same numbers, contiguous, one element behind an aligned address."""
    room = torch.zeros(t.numel() + 1, dtype=t.dtype, device=t.device)
    room.view(torch.uint8)[t.element_size():] = t.reshape(-1).view(torch.uint8)
    return room[1:].view(t.shape)


CALLS = ["rope_store_fp8", "attention_paged_fp8", "attention_decode_fp8", "attention_decode_fp8_rope", "attention_prefill_fp8"]


@pytest.mark.parametrize("name", CALLS)
def test_refusals(name):
    """Each wrong argument alone makes the call fail before anything is launched; the right ones pass."""
    op, good = getattr(ops(), name), good_call(name)
    rows = "qkv" if "qkv" in good else "q"
    out = "q_out" if "q_out" in good else "out"
    wrong = [dict(k_cache=good["k_cache"].view(torch.uint8)), dict(v_cache=good["v_cache"].to(BF)),
             dict(k_exp=good["k_exp"].to(torch.int32)), dict(k_cache=good["k_cache"][:, :, :32].contiguous()),
             dict(v_cache=good["v_cache"][:-1]), dict(v_exp=good["v_exp"][:, :, :3].contiguous()),
             dict(k_cache=good["k_cache"].transpose(1, 2).contiguous().transpose(1, 2)), dict(k_cache=good["k_cache"].cpu()),
             dict(block_table=good["block_table"].long()), dict(block_table=good["block_table"][0].contiguous()),
             dict(seq_slot=good["seq_slot"].float()), dict([(rows, good[rows].to(torch.float16))]),
             dict([(rows, good[rows][:, :-64].contiguous())]), dict([(rows, torch.cat([good[rows]] * 2, 1)[:, ::2])]),
             dict([(out, good[out][:1])]), dict([(out, good[out].float())]), dict(n_q=5), dict(n_q=0), dict(head_dim=32),
             dict(k_cache=shifted(good["k_cache"]))]
    if "seq_start" in good:
        wrong += [dict(cu_q=good["cu_q"][:2]), dict(seq_start=good["seq_start"][:1]), dict(max_q_len=0), dict(n_seqs=-1),
                  dict(seq_slot=good["seq_slot"][:1])]
    if "seq_kvlen" in good:
        wrong += [dict(seq_kvlen=good["seq_kvlen"][:1]), dict(seq_kvlen=good["seq_kvlen"].long()), dict(k_exp=shifted(good["k_exp"]))]
    if "table" in good:
        wrong += [dict(table=good["table"].to(BF)), dict(table=good["table"][:, :16].contiguous()), dict(table=good["table"][:0])]
    if "tok_pos" in good:
        wrong += [dict(tok_pos=good["tok_pos"][:1]), dict(tok_seq=good["tok_seq"].long())]
    if name == "attention_prefill_fp8":
        wrong += [dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(q=shifted(good["q"]))]
    before = [t.clone() for t in (good["k_cache"], good["v_cache"], good["k_exp"], good["v_exp"], good[out])]
    for w in wrong:
        with pytest.raises(ops().KernelError):
            op(**dict(good, **w))
    torch.cuda.synchronize()
    after = (good["k_cache"], good["v_cache"], good["k_exp"], good["v_exp"], good[out])
    assert all(same_bits(a, b) for a, b in zip(before, after))
    op(**good)
    torch.cuda.synchronize()


def test_exponents_at_any_address_where_the_call_takes_them():
    """Appends, the plain kernel and prompts read exponents byte by byte."""
    for name in ("rope_store_fp8", "attention_paged_fp8", "attention_prefill_fp8"):
        results = []
        for place in (lambda t: t, shifted):
            good = good_call(name)
            good["k_exp"], good["v_exp"] = place(good["k_exp"]), place(good["v_exp"])
            good["qkv" if "qkv" in good else "q"].fill_(0.25)
            out = getattr(ops(), name)(**good)
            results.append((out, good["k_exp"].clone(), good["v_exp"].clone(), good["k_cache"]))
        assert all(same_bits(a, b) for a, b in zip(*results)), name


@pytest.mark.parametrize("n_q,n_kv,hd", [(128, 1, 64), (128, 1, 128), (64, 1, 128)])
def test_prompt_of_the_widest_groups(n_q, n_kv, hd):
    starts, news = [0, 300, 60], [3, 2, 5]
    pc = filled([s + m for s, m in zip(starts, news)], n_kv, hd, seed=hd + n_q)
    q = torch.randn(sum(news), n_q * hd, generator=torch.Generator().manual_seed(1)).to(BF)
    out = prompt(pc, q, starts, news, n_q, n_kv, hd, hd ** -0.5, 0)
    check_prompt(pc, out, q, starts, news, n_q, n_kv, hd, hd ** -0.5, 0)


def test_many_sequences_in_a_step():
    """More sequences than a warp looks at in one go, most of them short, some empty, more items than thread blocks."""
    n_q, n_kv, hd = 8, 2, 64
    g = torch.Generator().manual_seed(9)
    lens = torch.randint(0, 90, (1500,), generator=g).tolist()
    pc = filled(lens, n_kv, hd, seed=9)
    n = len(lens)
    q = torch.randn(n, n_q * hd, generator=g).to(BF)
    out = torch.full((n, n_q * hd), math.nan, dtype=BF, device=DEV)
    ops().attention_decode_fp8(q.to(DEV), *pc.dev(), out, i32(pc.slots), i32(lens), pc.table.to(DEV), n_q, n_kv, hd, hd ** -0.5, 0, 90)
    two = torch.full((n, n_q * hd), math.nan, dtype=BF, device=DEV)
    some = [i for i, l in enumerate(lens) if l]
    ops().attention_prefill_fp8(q[some].to(DEV), *pc.dev(), two[:len(some)], i32(list(range(len(some) + 1))), i32([pc.slots[i] for i in some]),
                                i32([lens[i] - 1 for i in some]), pc.table.to(DEV), len(some), 1, n_q, n_kv, hd, hd ** -0.5)
    ops().check_tc_status(DEV)
    for row, i in enumerate(some):
        want, size = fp8_cache.attention(q[i:i + 1].double().view(1, n_q, hd), *pc.held(i, lens[i]), [lens[i] - 1], hd ** -0.5, 0)
        bound = allowed(want, size, BF, True)
        assert bool(((out[i].cpu().double().view(1, n_q, hd) - want).abs() <= bound).all()), i
        assert bool(((two[row].cpu().double().view(1, n_q, hd) - want).abs() <= bound).all()), i
    assert all(bool((out[i] == 0).all()) for i, l in enumerate(lens) if l == 0)
