"""The kernels of a cache in 8 bits at corners that their documentation allows, against tests/fp8_cache.py. Bounds: see test_cache_fp8_gpu.py."""
import pytest
import torch

import fp8_cache
from test_cache_fp8_gpu import BF, DEV, allowed, check_prompt, filled, good_call, i32, ops, prompt

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd,start,new,rows,max_pages", [(64, 4000, 64, 2048, 64), (128, 4216, 2, 2136, 67), (128, 4216, 2, 40000, 67),
                                                         (64, 4000, 64, 300, 64)])
def test_prompt_with_many_rows_behind_its_one_sequence(hd, start, new, rows, max_pages):
    """By its rows the step has more tiles of tokens than there are SMs, by its sequence few with many keys: how the work is cut has to
    fit the blocks and the scratch that the rows made the caller count on."""
    n_q, n_kv = (32, 8) if hd == 64 else (28, 4)
    pc = filled([start + new], n_kv, hd, seed=hd + new)
    table = torch.full((pc.table.shape[0], max_pages), pc.n_pages - 1, dtype=torch.int32)
    width = min(max_pages, pc.table.shape[1])
    table[:, :width] = pc.table[:, :width]
    q = torch.randn(rows, n_q * hd, generator=torch.Generator().manual_seed(1)).to(BF)
    for most in (new, rows):
        out = torch.full((rows, n_q * hd), 3.0, dtype=BF, device=DEV)
        ops().attention_prefill_fp8(q.to(DEV), *pc.dev(), out, i32([0, new]), i32(pc.slots), i32([start]), table.to(DEV), 1, most, n_q, n_kv,
                                    hd, hd ** -0.5)
        ops().check_tc_status(DEV)
        assert bool((out[new:] == 3.0).all())
        check_prompt(pc, out[:new].cpu().double(), q, [start], [new], n_q, n_kv, hd, hd ** -0.5, 0, rows=[0, 1, 17, 31, 32])


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("power", [116, 124, -100, -112, -126])
def test_queries_near_the_ends_of_their_range(hd, power):
    """Queries of 2^power with a scale that makes ordinary scores of them: half precision inside has room for every finite bfloat16. (2^-126:
    most are subnormal.)"""
    n_q, n_kv, starts, news = 8, 2, [150, 0], [40, 200]
    lens = [s + m for s, m in zip(starts, news)]
    pc = filled(lens, n_kv, hd, seed=5, spread=0.3)
    q = (torch.randn(sum(news), n_q * hd, generator=torch.Generator().manual_seed(3)) * 2.0 ** power).to(BF)
    assert bool(torch.isfinite(q).all()) and float(q.abs().max()) > 2.0 ** power
    scale = 2.0 ** (-power - 3)
    out = prompt(pc, q, starts, news, n_q, n_kv, hd, scale, 0)
    check_prompt(pc, out, q, starts, news, n_q, n_kv, hd, scale, 0, rows=[0, 1, 17, 100, 128])
    last = q[[news[0] - 1, sum(news) - 1]].contiguous()
    got = torch.empty_like(last, device=DEV)
    for max_len in (200, 0):
        ops().attention_decode_fp8(last.to(DEV), *pc.dev(), got, i32(pc.slots), i32(lens), pc.table.to(DEV), n_q, n_kv, hd, scale, 0, max_len)
        for i, l in enumerate(lens):
            want, size = fp8_cache.attention(last[i:i + 1].double().view(1, n_q, hd), *pc.held(i, l), [l - 1], scale, 0)
            bound = allowed(want, size, BF, True)
            err = (got[i].cpu().double().view(1, n_q, hd) - want).abs()
            assert bool((err <= bound).all()), float((err / bound).max())


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_large_queries_that_large_keys_are_orthogonal_to(hd, sign):
    """A block of keys near the largest number, queries as large, and products that are all zero: every score is 0, and an ordinary mean of
    the values comes out, although the factor of such a block's scores is beyond float32. (Prompts take no negative scale.)"""
    n_q, n_kv, l = 4, 2, 100
    g = torch.Generator().manual_seed(6)
    pc = fp8_cache.PlainCache([l], n_kv, hd, seed=4, nan_stale=True)
    k = torch.randn(l, n_kv, hd, generator=g)
    k[:, :, 1::2] = 0.0
    k[32:48] *= 1e37
    pc.append(0, 0, k, torch.randn(l, n_kv, hd, generator=g))
    q = torch.zeros(6, n_q, hd)
    q[:, :, 1::2] = torch.randn(6, n_q, hd // 2, generator=g) * 1e37
    q = q.reshape(6, -1).to(BF)
    if sign > 0:
        out = prompt(pc, q, [l - 6], [6], n_q, n_kv, hd, hd ** -0.5, 0)
        check_prompt(pc, out, q, [l - 6], [6], n_q, n_kv, hd, hd ** -0.5, 0)
    got = torch.empty(1, n_q * hd, dtype=BF, device=DEV)
    for max_len in (l, 0):
        ops().attention_decode_fp8(q[:1].to(DEV), *pc.dev(), got, i32(pc.slots), i32([l]), pc.table.to(DEV), n_q, n_kv, hd, sign * hd ** -0.5, 0,
                                   max_len)
        want, size = fp8_cache.attention(q[:1].double().view(1, n_q, hd), *pc.held(0, l), [l - 1], sign * hd ** -0.5, 0)
        assert bool(((got.cpu().double().view(1, n_q, hd) - want).abs() <= allowed(want, size, BF, True)).all())


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("pages", [1, 2, 3, 15])
@pytest.mark.parametrize("window", [0, 40, -48])
def test_prompts_longer_than_their_table(hd, pages, window):
    """Tokens behind the table's last page (a caller's mistake) see what one at its last position sees, as the plain kernel has it: no key
    that is not there, however many pages a step of the kernel has."""
    n_q, n_kv, room = 8, 2, 64 * pages
    starts, news = [room - 20, room + 30, max(room - 70, 0), 0], [40, 3, 90, room + 5]
    pc = filled([room + 64] * 4, n_kv, hd, seed=pages)
    table = pc.table[:, :pages].contiguous().to(DEV)
    q = torch.randn(sum(news), n_q * hd, generator=torch.Generator().manual_seed(2)).to(BF)
    cu = [sum(news[:i]) for i in range(5)]
    out = torch.full((sum(news), n_q * hd), float("nan"), dtype=BF, device=DEV)
    ops().attention_prefill_fp8(q.to(DEV), *pc.dev(), out, i32(cu), i32(pc.slots), i32(starts), table, 4, max(news), n_q, n_kv, hd,
                                hd ** -0.5, window)
    ops().check_tc_status(DEV)
    plain = torch.empty_like(out)
    pos = [s + j for s, m in zip(starts, news) for j in range(m)]
    ops().attention_paged_fp8(q.to(DEV), *pc.dev(), plain, i32(pos), i32([i for i, m in enumerate(news) for _ in range(m)]), i32(pc.slots),
                              table, n_q, n_kv, hd, hd ** -0.5, window)
    for i, (st, m) in enumerate(zip(starts, news)):
        k, v = pc.held(i, room)
        pick = sorted({0, m // 2, max(room - st - 1, 0), min(max(room - st, 0), m - 1), m - 1} & set(range(m)))
        want, size = fp8_cache.attention(q[cu[i]:cu[i] + m].double().view(m, n_q, hd)[pick], k, v, [min(st + r, room - 1) for r in pick],
                                         hd ** -0.5, window)
        for got, tensor_cores in ((out, True), (plain, False)):
            err = (got[cu[i]:cu[i] + m].cpu().double().view(m, n_q, hd)[pick] - want).abs()
            bound = allowed(want, size, BF, tensor_cores)
            assert bool((err <= bound).all()), (i, tensor_cores, float((err / bound).max()))


def test_a_window_as_wide_as_32_bits_is_no_window():
    """The kernel is chosen by what a window leaves to be read: with the widest one the same as without, to the bit."""
    n_q, n_kv, hd, lens = 8, 2, 64, [30000, 40]
    pc = filled(lens, n_kv, hd, seed=3, spread=0.2)
    q = torch.randn(2, n_q * hd, generator=torch.Generator().manual_seed(2)).to(BF).to(DEV)
    outs = []
    for window in (0, 2 ** 31 - 1, 30000, -2 ** 31 + 1):
        out = torch.empty_like(q)
        ops().attention_decode_fp8(q, *pc.dev(), out, i32(pc.slots), i32(lens), pc.table.to(DEV), n_q, n_kv, hd, hd ** -0.5, window, 30000)
        outs.append(out.cpu())
    assert all(torch.equal(o, outs[0]) for o in outs)


@pytest.mark.parametrize("n_q,n_kv,window", [(64, 4, 0), (64, 4, 100), (80, 2, 0), (64, 4, -100)])
def test_many_lanes_with_many_query_heads_and_room_for_a_million_positions(n_q, n_kv, window):
    """512 lanes over tables of 16,384 pages: the positions of their KV heads are counted, not those of their query heads."""
    hd, n, held = 64, 512, [1, 40, 70, 200]
    pc = filled(held, n_kv, hd, seed=1)
    table = torch.full((pc.table.shape[0], 16384), pc.n_pages - 1, dtype=torch.int32)
    table[:, :pc.table.shape[1]] = pc.table
    table, cache = table.to(DEV), pc.dev()
    who = [i % 4 for i in range(n)]
    q = torch.randn(n, n_q * hd, generator=torch.Generator().manual_seed(2)).to(BF)
    for max_len in (200, 0):
        out = torch.empty(n, n_q * hd, dtype=BF, device=DEV)
        ops().attention_decode_fp8(q.to(DEV), *cache, out, i32([pc.slots[i] for i in who]), i32([held[i] for i in who]), table, n_q, n_kv, hd,
                                   hd ** -0.5, window, max_len)
        for row in list(range(8)) + [255, 510, 511]:
            i = who[row]
            want, size = fp8_cache.attention(q[row:row + 1].double().view(1, n_q, hd), *pc.held(i, held[i]), [held[i] - 1], hd ** -0.5, window)
            bound = allowed(want, size, BF, True)
            assert bool(((out[row].cpu().double().view(1, n_q, hd) - want).abs() <= bound).all()), row


def test_a_step_beyond_32_bits_of_positions_is_refused():
    n_q = n_kv = 64
    hd, n = 64, 954
    pc = filled([3], n_kv, hd, seed=1)
    table = torch.zeros(pc.table.shape[0], 16384, dtype=torch.int32, device=DEV)
    table[:, :pc.table.shape[1]] = pc.table.to(DEV)
    q = torch.zeros(n, n_q * hd, dtype=BF, device=DEV)
    args = (i32(pc.slots * n), i32([3] * n), table, n_q, n_kv, hd, 0.125)
    cache = pc.dev()
    with pytest.raises(ops().KernelError, match="not supported"):
        ops().attention_decode_fp8(q, *cache, q, *args)
    ops().attention_decode_fp8(q, *cache, q, *args, 1000)             # as many as a window can touch are few
    torch.cuda.synchronize()


@pytest.mark.parametrize("name", ["attention_paged_fp8", "attention_prefill_fp8", "attention_decode_fp8"])
def test_tables_whose_positions_pass_32_bits_are_refused(name):
    """A table of 2^25 pages has room for 2^31 positions."""
    good = good_call(name)
    good["block_table"] = torch.zeros(1, 2 ** 25, dtype=torch.int32, device=DEV)
    good["seq_slot"].zero_()
    with pytest.raises(ops().KernelError, match="not supported|bad argument"):
        getattr(ops(), name)(**good)
    torch.cuda.synchronize()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("size", [1e26, 1e30, 1e37])
@pytest.mark.parametrize("back", [0.0, 90.0])
def test_values_of_very_different_size(hd, size, back):
    """A block of values near the largest numbers beside zeros, ordinary ones and tiny ones, seen alike or (back > 0) hardly at all: the others
    count in the softmax's denominator by their scores, whatever their values are. The block stands first, in the middle and last."""
    n_q, n_kv, new = 8, 2, 40
    lens = [100, 333, 1700, 1700]
    at = [0, 160, 1680, 32]
    g = torch.Generator().manual_seed(6)
    pc = fp8_cache.PlainCache(lens, n_kv, hd, seed=4, nan_stale=True)
    q = torch.randn(len(lens) * new, n_q, hd, generator=g) * 0.5
    q[:, :, 0] = 1.0
    for i, (l, p) in enumerate(zip(lens, at)):
        k, v = 0.5 * torch.randn(l, n_kv, hd, generator=g), torch.randn(l, n_kv, hd, generator=g)
        k[:, :, 0] = 0.0
        k[p:p + 16, :, 0] = -back * hd ** 0.5
        v[::2] *= 1e-3
        v[16 * (l // 48):] *= 1e-12
        v[16 * (l // 32):] = 0.0
        v[p:p + 16] = size * torch.randn(16, n_kv, hd, generator=g).clamp(-3, 3)
        pc.append(i, 0, k, v)
    q = q.reshape(len(lens) * new, -1).to(BF)
    cache, table, scale = pc.dev(), pc.table.to(DEV), hd ** -0.5
    starts = [l - new for l in lens]
    # prompts: all sequences in a call, and each alone (in turns and in runs where it is long); tiles of 128 / 4 tokens and more
    for news in ([new] * 4, [7, 7, 7, 7]):
        pick = [i * new + j for i, m in enumerate(news) for j in range(m)]
        rows = [0, 1, 6, 20, 39]
        out = prompt(pc, q[pick], starts, news, n_q, n_kv, hd, scale, 0, cache)
        check_prompt(pc, out, q[pick], starts, news, n_q, n_kv, hd, scale, 0, rows=rows)
    for i in range(4):
        mine = q[i * new:(i + 1) * new]
        out = torch.empty(new, n_q * hd, dtype=BF, device=DEV)
        ops().attention_prefill_fp8(mine.to(DEV), *cache, out, i32([0, new]), i32(pc.slots[i:i + 1]), i32(starts[i:i + 1]), table, 1, new, n_q,
                                    n_kv, hd, scale)
        want, size_ = fp8_cache.attention(mine.double().view(new, n_q, hd)[[0, 20, 39]], *pc.held(i, lens[i]),
                                          [starts[i] + r for r in (0, 20, 39)], scale, 0)
        err = (out.cpu().double().view(new, n_q, hd)[[0, 20, 39]] - want).abs()
        assert bool((err <= allowed(want, size_, BF, True)).all()), i
    last = q[new - 1::new].contiguous()
    got = torch.empty_like(last, device=DEV)
    for max_len in (1700, 0):
        for pick in ([0, 1, 2, 3], [0], [2], [3]):
            part = torch.empty(len(pick), n_q * hd, dtype=BF, device=DEV)
            ops().attention_decode_fp8(last[pick].to(DEV), *cache, part, i32([pc.slots[i] for i in pick]), i32([lens[i] for i in pick]), table,
                                       n_q, n_kv, hd, scale, 0, max_len)
            got[pick] = part
            for i in pick:
                want, size_ = fp8_cache.attention(last[i:i + 1].double().view(1, n_q, hd), *pc.held(i, lens[i]), [lens[i] - 1], scale, 0)
                err = (got[i].cpu().double().view(1, n_q, hd) - want).abs()
                bound = allowed(want, size_, BF, True)
                assert bool((err <= bound).all()), (i, max_len, float((err / bound).max()))
    plain = torch.empty_like(got)
    ops().attention_paged_fp8(last.to(DEV), *cache, plain, i32([l - 1 for l in lens]), i32([0, 1, 2, 3]), i32(pc.slots), table, n_q, n_kv, hd,
                              scale)
    for i in range(4):
        want, size_ = fp8_cache.attention(last[i:i + 1].double().view(1, n_q, hd), *pc.held(i, lens[i]), [lens[i] - 1], scale, 0)
        assert bool(((plain[i].cpu().double().view(1, n_q, hd) - want).abs() <= allowed(want, size_, BF, False)).all())


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("size", [1e26, 1e30, 1e37])
@pytest.mark.parametrize("back", [0.0, 90.0])
def test_values_of_very_different_size(hd, size, back):
    """A block of values near the largest numbers beside zeros, ordinary ones and tiny ones, seen alike or (back > 0) hardly at all: the others
    count in the softmax's denominator by their scores, whatever their values are. The block stands first, in the middle and last."""
    n_q, n_kv, new = 8, 2, 40
    lens = [100, 333, 1700, 1700]
    at = [0, 160, 1680, 32]
    g = torch.Generator().manual_seed(6)
    pc = fp8_cache.PlainCache(lens, n_kv, hd, seed=4, nan_stale=True)
    q = torch.randn(len(lens) * new, n_q, hd, generator=g) * 0.5
    q[:, :, 0] = 1.0
    for i, (l, p) in enumerate(zip(lens, at)):
        k, v = 0.5 * torch.randn(l, n_kv, hd, generator=g), torch.randn(l, n_kv, hd, generator=g)
        k[:, :, 0] = 0.0
        k[p:p + 16, :, 0] = -back * hd ** 0.5
        v[::2] *= 1e-3
        v[16 * (l // 48):] *= 1e-12
        v[16 * (l // 32):] = 0.0
        v[p:p + 16] = size * torch.randn(16, n_kv, hd, generator=g).clamp(-3, 3)
        pc.append(i, 0, k, v)
    q = q.reshape(len(lens) * new, -1).to(BF)
    cache, table, scale = pc.dev(), pc.table.to(DEV), hd ** -0.5
    starts = [l - new for l in lens]
    # prompts: all sequences in a call, and each alone (in turns and in runs where it is long); tiles of 128 / 4 tokens and more
    for news in ([new] * 4, [7, 7, 7, 7]):
        pick = [i * new + j for i, m in enumerate(news) for j in range(m)]
        rows = [0, 1, 6, 20, 39]
        out = prompt(pc, q[pick], starts, news, n_q, n_kv, hd, scale, 0, cache)
        check_prompt(pc, out, q[pick], starts, news, n_q, n_kv, hd, scale, 0, rows=rows)
    for i in range(4):
        mine = q[i * new:(i + 1) * new]
        out = torch.empty(new, n_q * hd, dtype=BF, device=DEV)
        ops().attention_prefill_fp8(mine.to(DEV), *cache, out, i32([0, new]), i32(pc.slots[i:i + 1]), i32(starts[i:i + 1]), table, 1, new, n_q,
                                    n_kv, hd, scale)
        want, size_ = fp8_cache.attention(mine.double().view(new, n_q, hd)[[0, 20, 39]], *pc.held(i, lens[i]),
                                          [starts[i] + r for r in (0, 20, 39)], scale, 0)
        err = (out.cpu().double().view(new, n_q, hd)[[0, 20, 39]] - want).abs()
        assert bool((err <= allowed(want, size_, BF, True)).all()), i
    last = q[new - 1::new].contiguous()
    got = torch.empty_like(last, device=DEV)
    for max_len in (1700, 0):
        for pick in ([0, 1, 2, 3], [0], [2], [3]):
            part = torch.empty(len(pick), n_q * hd, dtype=BF, device=DEV)
            ops().attention_decode_fp8(last[pick].to(DEV), *cache, part, i32([pc.slots[i] for i in pick]), i32([lens[i] for i in pick]), table,
                                       n_q, n_kv, hd, scale, 0, max_len)
            got[pick] = part
            for i in pick:
                want, size_ = fp8_cache.attention(last[i:i + 1].double().view(1, n_q, hd), *pc.held(i, lens[i]), [lens[i] - 1], scale, 0)
                err = (got[i].cpu().double().view(1, n_q, hd) - want).abs()
                bound = allowed(want, size_, BF, True)
                assert bool((err <= bound).all()), (i, max_len, float((err / bound).max()))
    plain = torch.empty_like(got)
    ops().attention_paged_fp8(last.to(DEV), *cache, plain, i32([l - 1 for l in lens]), i32([0, 1, 2, 3]), i32(pc.slots), table, n_q, n_kv, hd,
                              scale)
    for i in range(4):
        want, size_ = fp8_cache.attention(last[i:i + 1].double().view(1, n_q, hd), *pc.held(i, lens[i]), [lens[i] - 1], scale, 0)
        assert bool(((plain[i].cpu().double().view(1, n_q, hd) - want).abs() <= allowed(want, size_, BF, False)).all())


@pytest.mark.parametrize("hd", [64, 128])
def test_values_of_very_different_size_in_a_long_prompt(hd):
    """300 tokens behind 12,000: many rows whose denominators are taken once more, over many keys, while the rest of the block waits."""
    n_q, n_kv, start, new = 8, 2, 12000, 300
    l = start + new
    g = torch.Generator().manual_seed(7)
    pc = fp8_cache.PlainCache([l], n_kv, hd, seed=4)
    v = torch.randn(l, n_kv, hd, generator=g)
    v[::7] = 0.0
    v[64:96] = 0.0
    v[96:112] *= 1e30
    pc.append(0, 0, torch.randn(l, n_kv, hd, generator=g), v)
    q = (0.3 * torch.randn(new, n_q * hd, generator=g)).to(BF)
    out = prompt(pc, q, [start], [new], n_q, n_kv, hd, hd ** -0.5, 0)
    want, size = fp8_cache.attention(q.double().view(new, n_q, hd)[[0, 150, 299]], *pc.held(0, l), [start + r for r in (0, 150, 299)],
                                     hd ** -0.5, 0)
    # 12,300 keys: eight times the keys that `allowed` counts float32 sums for
    bound = allowed(want, size, BF, True) + 2.0 ** -10 * size
    assert bool(((out.view(new, n_q, hd)[[0, 150, 299]] - want).abs() <= bound).all())


@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("hd", [48, 64, 128])
def test_sums_of_the_largest_values(hd, dtype):
    """Values near the largest number that a block can hold, many of them: their mean is one of them. Tiny ones beside them in other heads."""
    n_q, n_kv, l = 4, 2, 700
    g = torch.Generator().manual_seed(3)
    pc = fp8_cache.PlainCache([l], n_kv, hd, seed=4)
    v = torch.randn(l, n_kv, hd, generator=g) * 1e-15
    v[:, 0] = 3e38
    v[:, 0, 1] = -1e38
    pc.append(0, 0, 0.1 * torch.randn(l, n_kv, hd, generator=g), v)
    q = torch.randn(1, n_q * hd, generator=g).to(dtype)
    want, size = fp8_cache.attention(q.double().view(1, n_q, hd), *pc.held(0, l), [l - 1], hd ** -0.5, 0)
    outs = []
    plain = torch.empty_like(q, device=DEV)
    ops().attention_paged_fp8(q.to(DEV), *pc.dev(), plain, i32([l - 1]), i32([0]), i32(pc.slots), pc.table.to(DEV), n_q, n_kv, hd, hd ** -0.5)
    outs.append((plain, False))
    if dtype is BF and hd != 48:
        for max_len in (l, 0):
            out = torch.empty_like(plain)
            ops().attention_decode_fp8(q.to(DEV), *pc.dev(), out, i32(pc.slots), i32([l]), pc.table.to(DEV), n_q, n_kv, hd, hd ** -0.5, 0, max_len)
            outs.append((out, True))
        outs.append((prompt(pc, q, [l - 1], [1], n_q, n_kv, hd, hd ** -0.5, 0), True))
    for out, tensor_cores in outs:
        err = (out.cpu().double().view(1, n_q, hd) - want).abs()
        bound = allowed(want, size, dtype, tensor_cores)
        assert bool((err <= bound).all()), (tensor_cores, float((err / bound).max()))


@pytest.mark.parametrize("window", [0, 1, 40, -1, -2, -3, -64])
def test_positions_below_zero_see_no_key(window):
    """A lane without a sequence, in the plain kernel: zeros, whatever the window or chunk, and nothing in front of its page is read."""
    n_q, n_kv, hd, pos = 4, 2, 64, [-1, -2, -6, -64, 5]
    pc = filled([20], n_kv, hd, seed=1, nan_stale=False)
    pc.table[pc.slots[0], 0] = 0                       # the first page that there is: before it is nothing
    q = torch.randn(len(pos), n_q * hd, generator=torch.Generator().manual_seed(1)).to(BF)
    out = torch.full((len(pos), n_q * hd), float("nan"), dtype=BF, device=DEV)
    ops().attention_paged_fp8(q.to(DEV), *pc.dev(), out, i32(pos), i32([0] * len(pos)), i32(pc.slots), pc.table.to(DEV), n_q, n_kv, hd, 0.125,
                              window)
    assert bool((out[:4] == 0).all())
    want, size = fp8_cache.attention(q[4:].double().view(1, n_q, hd), *pc.held(0, 20), [5], 0.125, window)
    assert bool(((out[4:].cpu().double().view(1, n_q, hd) - want).abs() <= allowed(want, size, BF, False)).all())
