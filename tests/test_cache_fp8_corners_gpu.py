"""The kernels of a cache in 8 bits at corners that their documentation allows, against tests/fp8_cache.py. Bounds: see test_cache_fp8_gpu.py."""
import math

import pytest
import torch

import fp8_cache
from fp8_cache import F8, PlainCache
from test_cache_fp8_gpu import BF, DEV, F32, allowed, angles, check_cache, check_prompt, filled, i32, ops, plain_store, prompt, same_bits, store

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
