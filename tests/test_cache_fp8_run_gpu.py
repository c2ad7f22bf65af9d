"""The operators of a cache in 8 bits together, as layers and engines run them: prompts in pieces and steps of one token through
the attention part, whole engines against the plain model with its keys and values held in 8 bits, captured steps."""
import json
import math
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import fp8_cache
import helpers
import plain_llama as plain
from test_cache_fp8_gpu import allowed, same_bits
from test_parts_gpu import DTYPES, build, kernel_plan, make_ctx

pytestmark = pytest.mark.gpu
DEV = "cuda"
F8 = torch.float8_e4m3fn


class Seen:
    """The projections of a layer, kept for the test."""

    def __init__(self, linear):
        self.linear, self.weight, self.rows = linear, linear.weight, None

    def __call__(self, x):
        self.rows = self.linear(x)
        return self.rows


class AsItComes:
    """In place of the projection behind the attention."""

    def __call__(self, x):
        return x


def layer(dtype, n_q, n_kv, hd, window, position):
    from llm_infer_engine_b200.config import PartSpec
    spec = PartSpec("rope", {"rot_dim": hd, "theta": 10000.0, "scaling": None}) if position else PartSpec("none", {})
    mixer, _ = build("mixer", "gqa_attention", {"hidden": 96, "n_heads": n_q, "n_kv_heads": n_kv, "head_dim": hd, "window": window,
                                                "scale": None, "position": spec}, dtype, seed=6, std=0.15)
    mixer.qkv, mixer.o = Seen(mixer.qkv), AsItComes()
    return mixer


class Mirror(fp8_cache.PlainCache):
    """A plain cache that has a unit's pages and tables as they are now."""

    def __init__(self, kv, slots):
        self.k, self.v, self.ke, self.ve = kv.k.cpu(), kv.v.cpu(), kv.k_exp.cpu(), kv.v_exp.cpu()
        self.table, self.slots = kv.block_table.cpu(), slots
        self.n_kv, self.hd = kv.k.shape[1], kv.k.shape[3]


def lost(v):
    """What half precision's smallest steps take from weights far below a row's largest, where `allowed` counts relative steps only
    (scores here lie up to 500 apart). A weight that goes into a product of codes is w_j = 2^(s_j + e_j - R + 7), e_j the exponent of
    the value's block, R at most the row's largest s + e, which key m has; below 2^-14 it is off by 2^-25. The row's error is at most
    sum_j 2^-25 |code_j| 2^(R - 7) / 2^(s_m) <= n 2^-25 448 2^(e_m - 7), and 448 2^(e_m) is less than twice its block's largest
    value: n 2^-31 max |v|."""
    return v.shape[0] * 2.0 ** -31 * float(v.abs().max())


@pytest.mark.parametrize("dtype,n_q,n_kv,hd,window,position", [
    ("bfloat16", 8, 2, 64, 0, True), ("bfloat16", 8, 8, 128, 0, True), ("bfloat16", 14, 2, 64, 100, True),
    ("bfloat16", 40, 2, 64, 0, True), ("bfloat16", 8, 2, 128, 100, False), ("bfloat16", 6, 3, 32, 50, True),
    ("float32", 4, 2, 64, 0, True), ("float32", 3, 1, 80, 70, False)])
def test_a_layer_by_pieces_and_tokens(dtype, n_q, n_kv, hd, window, position):
    """Prompts in one, two and three pieces, some beside steps of one token, then steps of one token for all: after every step the
    pages hold bit for bit what the plain form makes of the projections, and the output is the plain attention over the pages.
    With a window, pages that no later token reads are given back and go to others."""
    from llm_infer_engine_b200.cache import Cache
    T = DTYPES[dtype]
    mixer = layer(dtype, n_q, n_kv, hd, window, position)
    cache = Cache([mixer.cache_requests()], 4, 64 * 18, 512, T, DEV, F8)
    unit, plan = cache.unit(0), kernel_plan(dtype)
    slots = [cache.take_slot() for _ in range(3)]
    held = [0, 0, 0]
    g = torch.Generator().manual_seed(7)
    tensor_cores = dtype == "bfloat16" and hd in (64, 128)
    for step, news in enumerate([(5, 130, 40), (1, 61, 3), (1, 1, 70), (1, 1, 1), (1, 1, 1), (200, 1, 15), (1, 1, 1), (1, 1, 1)]):
        x = torch.randn(sum(news), 96, generator=g) * torch.exp(torch.randn(sum(news), 1, generator=g))
        for s, h, m in zip(slots, held, news):
            cache.reserve(s, h + m)
        mirror = Mirror(unit.kv, slots)
        y = mixer.forward(x.to(DEV, T), make_ctx(list(news), held, slots, dtype, plan), unit, True).cpu()
        qkv = mixer.qkv.rows.cpu().float().view(sum(news), n_q + 2 * n_kv, hd)
        table = mixer.position.table.cpu() if position else None
        row = 0
        for i, (h, m) in enumerate(zip(held, news)):
            mine = qkv[row:row + m]
            turned = fp8_cache.rotate(mine[:, :n_q + n_kv], table[h:h + m], hd) if position else mine[:, :n_q + n_kv]
            mirror.append(i, h, turned[:, n_q:], mine[:, n_q + n_kv:])
            k, v = mirror.held(i, h + m)
            want, size = fp8_cache.attention(turned[:, :n_q].to(T).double(), k, v, list(range(h, h + m)), hd ** -0.5, window)
            err = (y[row:row + m].double().view(m, n_q, hd) - want).abs()
            bound = allowed(want, size, T, tensor_cores) + (lost(v) if tensor_cores else 0.0)
            assert bool((err <= bound).all()), (step, i, float((err / bound).max()))
            row += m
            cache.note_appended(slots[i], h + m, device_updated=False)
        pages = unit.kv.k.shape[0] - 1             # the last one belongs to nobody
        assert torch.equal(unit.kv.k_exp.cpu()[:pages], mirror.ke[:pages]) and torch.equal(unit.kv.v_exp.cpu()[:pages], mirror.ve[:pages]), step
        assert same_bits(unit.kv.k.cpu()[:pages], mirror.k[:pages]) and same_bits(unit.kv.v.cpu()[:pages], mirror.v[:pages]), step
        held = [h + m for h, m in zip(held, news)]
    if dtype == "bfloat16":
        from llm_infer_engine_b200.kernels import ops
        ops.check_tc_status(DEV)
    for s in slots:
        cache.give_back_slot(s)
    cache.check()


# ------------------------------------------------------------------------------------------ engines
def in_8_bits(x):
    """Keys or values [heads, T, hd] of a sequence that came in one step, as the cache holds them."""
    y = x.clone()
    for h in range(x.shape[0]):
        for b in range(0, x.shape[1], fp8_cache.BLOCK):
            part = x[h, b:b + fp8_cache.BLOCK]
            e = fp8_cache.exponent_of(part)
            y[h, b:b + fp8_cache.BLOCK] = fp8_cache.to_codes(part, e).float() * 2.0 ** e
    return y


@pytest.fixture
def plain_in_8_bits(monkeypatch):
    whole = plain.causal_gqa_attention

    def switch(on):
        monkeypatch.setattr(plain, "causal_gqa_attention",
                            (lambda q, k, v: whole(q, in_8_bits(k), in_8_bits(v))) if on else whole)
    return switch


def rms(x):
    return float(x.double().square().mean().sqrt())


@pytest.mark.parametrize("tag", ["a", "b", "c"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_engine_against_the_plain_model(plain_in_8_bits, dtype, tag):
    """Prompts of one step each. What the engine may differ by from the plain model with keys and values in 8 bits: its own
    rounding, and numbers that this puts on the other side of the middle between two codes, each a step off. In float32 (relative
    error 1e-6 against steps of 2^-4 and more) that is at most one number in ten thousand, against all of them rounded by 0.29 of a step: a few
    hundredths of what the 8 bits themselves make (bound: a tenth). In bfloat16 one number in eight at most goes over (2^-8 / 2^-4 and
    the block's smaller ones never more): sqrt(1/8) / 0.29, as much as the 8 bits themselves make and a quarter more (bound: twice)."""
    from llm_infer_engine_b200 import Engine
    folder = helpers.model_folder(tag)
    w, cfg = helpers.plain_weights(folder), helpers.read_config(folder)
    lens = [n for n in (1, 16, 17, 63, 100, 128) if n <= cfg["max_position_embeddings"]]
    requests = {f"r{i}": helpers.random_tokens(cfg["vocab_size"], n, seed=300 + i) for i, n in enumerate(lens)}
    engine = Engine(folder, dtype=dtype, max_batch=8, max_tokens=64 * 40, cuda_graph=False, cache_dtype="float8_e4m3")
    assert engine.cache.kv_dtype == F8 and engine.cache_dtype == F8
    got = helpers.run_plan_engine(engine, helpers.plan_whole(requests))
    whole, eight = {}, {}
    for r, toks in requests.items():
        plain_in_8_bits(False)
        whole[r] = plain.logits(w, cfg, toks)
        plain_in_8_bits(True)
        eight[r] = plain.logits(w, cfg, toks)
    apart = torch.cat([got[r] - eight[r] for r in requests])
    made = torch.cat([whole[r] - eight[r] for r in requests])
    assert rms(made) > 0
    own = helpers.logit_bound(dtype, torch.cat(list(eight.values())))
    assert rms(apart) <= (0.1 if dtype == "float32" else 2.0) * rms(made) + own, (rms(apart), rms(made), own)
    engine.cache.check()
    assert engine.cache.free_pages() == engine.cache.n_pages


@pytest.mark.parametrize("tag,dtype", [("a", "float32"), ("c", "float32"), ("b", "bfloat16"), ("c", "bfloat16")])
def test_captured_generation_is_eager_generation(tag, dtype):
    """More requests than slots, prompts of several lengths, generation past block and page borders: with captured steps and
    without, the same tokens; and the cache takes what it says."""
    from llm_infer_engine_b200 import Engine, generate
    folder = helpers.model_folder(tag)
    cfg = helpers.read_config(folder)
    prompts = [helpers.random_tokens(cfg["vocab_size"], n, seed=400 + i) for i, n in enumerate([5, 60, 17, 3, 40, 1, 63])]
    out = {}
    for graph in (False, True):
        engine = Engine(folder, dtype=dtype, max_batch=3, max_tokens=64 * 9, cuda_graph=graph, cache_dtype="float8_e4m3")
        out[graph] = [generate(engine, prompts, max_new_tokens=30, stop_ids=[]) for _ in range(2)]
        kv = cfg["num_hidden_layers"] * cfg["num_key_value_heads"]
        assert engine.kv_bytes_per_token() == kv * 2 * cfg["head_dim"] + math.ceil(2 * kv / 16)
        engine.cache.check()
        assert engine.cache.free_slots() == 3 and engine.cache.free_pages() == engine.cache.n_pages
    assert out[False] == out[True]
    assert out[True][0] == out[True][1]            # pages that had other owners make no difference
    assert all(len(o) == 30 for o in out[True][0])


@pytest.mark.parametrize("which", ["zemivik", "burinex", "rogizen", "selinex"])
def test_models_whose_mixers_do_not_know_it_are_refused(which, tmp_path):
    import importlib
    from llm_infer_engine_b200 import Engine, EngineError, write_random_model
    cfg = importlib.import_module("plain_zemivik").TINY_A if which == "zemivik" else importlib.import_module(f"test_{which}_host").CFG
    write_random_model(cfg, str(tmp_path), seed=1)
    with pytest.raises(EngineError, match="8 bits"):
        Engine(str(tmp_path), max_batch=2, max_seq_len=64, cache_dtype="float8_e4m3")
    Engine(str(tmp_path), max_batch=2, max_seq_len=64, cuda_graph=False)


@pytest.mark.parametrize("which", ["a join with nothing to join", "a join", "one launch", "prompt", "prompt in runs", "append"])
def test_the_kernel_behind_reads_finished_rows(which):
    """Launches that may begin early, bit for bit as launches that may not: what a call leaves goes straight into the next kernel,
    forty times through the same buffer."""
    from llm_infer_engine_b200.kernels import ops
    n_q, n_kv, hd = 16, 4, 128
    n, held = {"a join with nothing to join": (111, 1920), "a join": (5, 9000), "one launch": (12, 300), "prompt": (40, 90),
               "prompt in runs": (6, 3000), "append": (40, 90)}[which]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)                                # noqa: E731
    pages = -(-held // 64)
    shape = (n * pages, n_kv, 64, hd)
    g = torch.Generator(device=DEV).manual_seed(1)
    k, v = (torch.randint(0, 120, shape, generator=g, device=DEV).to(torch.uint8).view(F8) for _ in range(2))
    exps = torch.full(shape[:2] + (4,), -7, dtype=torch.int8, device=DEV)
    table = torch.arange(n * pages, dtype=torch.int32, device=DEV).view(n, pages)
    slots, lens, starts, cu = i32(list(range(n))), i32([held] * n), i32([held - 1] * n), i32(list(range(n + 1)))
    qs = torch.randn(40, n, n_q * hd, generator=g, device=DEV).to(torch.bfloat16)

    def run():
        buf, half, outs = torch.zeros(n, n_q * hd, dtype=torch.bfloat16, device=DEV), torch.empty_like(qs[0][:, :8 * hd]), []
        half, cache = half.contiguous(), [t.clone() for t in (k, v, exps, exps)]
        for q in qs:
            if which.startswith("prompt"):
                ops.attention_prefill_fp8(q, k, v, exps, exps, buf, cu, slots, starts, table, n, 1, n_q, n_kv, hd, hd ** -0.5)
            elif which == "append":
                ops.rope_store_fp8(q, half, *cache, None, cu, slots, starts, table, n, 1, 8, n_kv, hd, 0)
                ops.attention_decode_fp8(q, *cache, buf, slots, lens, table, n_q, n_kv, hd, hd ** -0.5, 0, held)
            else:
                ops.attention_decode_fp8(q, k, v, exps, exps, buf, slots, lens, table, n_q, n_kv, hd, hd ** -0.5, 0, held)
            outs.append(torch.empty(n, 8 * hd, dtype=torch.bfloat16, device=DEV))
            ops.rope_store_fp8(buf, outs[-1], k, v, exps, exps, None, cu, slots, starts, table, n, 1, 8, n_kv, hd, 0, False)
        torch.cuda.synchronize()
        return torch.stack(outs)

    early = [run() for _ in range(3)]
    ops.set_pdl(False)
    try:
        late = run()
    finally:
        ops.set_pdl(True)
    for e in early:
        assert torch.equal(e, late)


def test_options_that_do_not_go_together():
    from llm_infer_engine_b200 import Engine, EngineError
    folder = helpers.model_folder("c")
    with pytest.raises(EngineError, match="split"):
        Engine(folder, max_batch=2, cache_dtype="float8_e4m3", decode_attention="split")
    with pytest.raises(EngineError, match="cache_dtype"):
        Engine(folder, max_batch=2, cache_dtype="int8")


def test_programs(tmp_path):
    """The command line and the replay program with their cache's type named: what the engine gives."""
    from llm_infer_engine_b200 import Engine, generate
    folder = helpers.model_folder("c")
    cfg = helpers.read_config(folder)
    prompt = helpers.random_tokens(cfg["vocab_size"], 70, seed=500)
    engine = Engine(folder, dtype="float32", max_batch=4, max_tokens=64 * 12, cuda_graph=False, cache_dtype="float8_e4m3")
    run = subprocess.run([sys.executable, os.path.join(helpers.ROOT, "main.py"), "--model", folder, "--prompt-ids",
                          ",".join(map(str, prompt)), "--dtype", "float32", "--cache-dtype", "float8_e4m3", "--env-file",
                          str(tmp_path / "none")], capture_output=True, text=True, timeout=300,
                         env=dict(os.environ, LLM_MAX_NEW_TOKENS="6"))
    assert run.returncode == 0, run.stderr[-2000:]
    assert "cache float8_e4m3" in run.stdout
    ids = [int(x) for x in run.stdout.split("OUTPUT")[1].split("=" * 70)[1].split()]
    assert ids == generate(engine, [prompt], max_new_tokens=6)[0]

    steps = helpers.plan_batched({"x": prompt, "y": prompt[:21]}, batch_size=2)
    want = helpers.run_plan_engine(engine, steps)
    run = subprocess.run([sys.executable, os.path.join(helpers.ROOT, "bin", "trace_run"), "--model", folder, "--dtype", "float32",
                          "--out", str(tmp_path), "--max-tokens", str(helpers.max_tokens_for(steps)), "--cache-dtype", "float8_e4m3"],
                         input="\n".join(json.dumps(s) for s in steps) + "\n", capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]
    last = [s for s in steps if any(e["want"] for e in s["entries"])][-1]
    rows = torch.from_numpy(np.fromfile(str(tmp_path / f"{last['step']}.f32"), dtype="<f4").reshape(-1, cfg["vocab_size"]).copy())
    end = torch.cat([want[e["id"]][-len(e["want"]):] for e in last["entries"] if e["want"]])
    assert torch.equal(rows, end)
