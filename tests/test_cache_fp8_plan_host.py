"""Attention of prompts over a cache in 8 bits: the host counts thread blocks and scratch before it knows the lengths, the device cuts the
work by the lengths that are there. The two have to agree: here the host's count (asked of the library) against the device's arithmetic,
restated."""
import ctypes
import random

import pytest

SMS, LEAST, WHOLE = 148, 256, 768


@pytest.fixture(scope="module")
def host_plan():
    from llm_infer_engine_b200.kernels import build
    f = build.load("attention_prefill_fp8").llmie_attention_prefill_fp8_plan
    f.argtypes = [ctypes.c_int] * 8 + [ctypes.POINTER(ctypes.c_longlong)]
    f.restype = ctypes.c_int

    def plan(n_tokens, n_seqs, max_q_len, max_pages, n_q, n_kv, hd, window):
        out = (ctypes.c_longlong * 4)()
        assert f(n_tokens, n_seqs, max_q_len, max_pages, n_q, n_kv, hd, window, out) == 0
        return list(out)

    return plan


def first_visible(pos, window):
    return max(pos - window + 1, 0) if window > 0 else pos - pos % -window if window < 0 else 0


def device_cut(run, starts, news, max_q_len, max_pages, n_q, n_kv, hd, window):
    """Pieces of work and partial results of a step: what the blocks find by the lengths. `run`: what the host hands over (0: whole)."""
    keys = 128 if hd == 64 else 64
    tok_x = 128 // (n_q // n_kv)
    tok = tok_x if max_q_len <= tok_x else 2 * tok_x

    def tiles_of(start, t0, n):
        lo = first_visible(min(start + t0, max_pages * 64 - 1), window) // keys
        return max((min(start + t0 + n, max_pages * 64) - 1) // keys - lo + 1, 0)

    seqs = []                                                 # tiles of tokens, key tiles of the first and the last of them
    for start, new in zip(starts, news):
        tiles = -(-new // tok)
        if tiles:
            seqs.append((tiles, tiles_of(start, 0, min(tok, new)), tiles_of(start, (tiles - 1) * tok, new - (tiles - 1) * tok)))

    def parts(last, r):
        return max(1, (last - r - 1) // -r) if r < 0 else max(1, (last + r // 2) // r)

    def chosen():
        if run == 0 or max((last for _, _, last in seqs), default=0) <= WHOLE // keys:
            return 1 << 30
        share = sum(t * (f + l) for t, f, l in seqs) * n_kv / SMS
        up = -int(-share // 1)
        most = max(run, LEAST // keys, up)
        if sum(t for t, _, _ in seqs) * n_kv > SMS:
            return most
        r = max(run, LEAST // keys, -int(-(share / 2) // 1))
        for _ in range(24):
            if sum(t * parts(l, -r) for t, _, l in seqs) * n_kv <= SMS:
                return -r
            r += (r + 7) // 8
        return most

    r = chosen()
    pieces = sum(t * parts(l, r) for t, _, l in seqs) * n_kv
    results = sum(t * parts(l, r) for t, _, l in seqs if parts(l, r) > 1) * n_kv
    return pieces, results


def check(host_plan, starts, news, rows, max_q_len, max_pages, n_q, n_kv, hd, window):
    run, cut, blocks, room = host_plan(rows, len(news), max_q_len, max_pages, n_q, n_kv, hd, window)
    pieces, results = device_cut(run, starts, news, max_q_len, max_pages, n_q, n_kv, hd, window)
    what = (starts, news, rows, max_q_len, max_pages, n_q, n_kv, hd, window, run, cut, blocks, pieces, results)
    assert pieces <= blocks, what
    assert results <= (room if cut else 0), what


def test_a_step_with_many_rows_behind_its_one_sequence(host_plan):
    """2,048 rows of which 64 belong to a sequence: many tiles by the rows, few by the lengths."""
    for most in (64, 2048):
        check(host_plan, [4000], [64], 2048, most, 64, 32, 8, 64, 0)
    check(host_plan, [65000], [64], 8192, 64, 1100, 32, 8, 128, 0)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("padded", [False, True])
def test_cuts_have_room(host_plan, hd, padded):
    """Steps of all kinds, with as many rows as the sequences bring and with more."""
    rng = random.Random(hd + padded)

    def between(lo, hi):
        return int(round(2 ** rng.uniform(0, 1) * lo * (hi / lo) ** rng.random())) if rng.random() < 0.9 else lo

    for _ in range(4000):
        n_kv = rng.choice([1, 2, 4, 8, 16])
        n_q = n_kv * rng.choice([1, 2, 3, 4, 7, 8, 16, 64, 128])
        n = between(1, 200)
        longest = between(1, 3000)
        news = [rng.randint(0, longest) if rng.random() < 0.5 else min(longest, rng.randint(1, 9)) for _ in range(n)]
        starts = [between(1, 60000) if rng.random() < 0.7 else 0 for _ in range(n)]
        if not sum(news):
            continue
        rows = sum(news) + (between(1, 40000) if padded else 0)
        max_q_len = max(news) if rng.random() < 0.8 else min(rows, max(news) + between(1, 500))
        need = -(-max(s + m for s, m in zip(starts, news)) // 64)
        max_pages = need if rng.random() < 0.5 else between(need, 4 * need) if rng.random() < 0.8 else max(1, need // 2)
        window = rng.choice([0, 0, 0, between(1, 20000), -between(1, 20000)])
        check(host_plan, starts, news, rows, max_q_len, max_pages, n_q, n_kv, hd, window)
