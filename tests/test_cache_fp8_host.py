"""The cache in 8 bits where no GPU is needed: its storage, who may use it, the names it goes by, calls that are refused."""
import pytest
import torch

import fp8_cache
from llm_infer_engine_b200 import EngineError
from llm_infer_engine_b200.cache import Cache, KVRequest
from llm_infer_engine_b200.engine.engine import resolve_cache_dtype
from llm_infer_engine_b200.kernels import ops

F8 = torch.float8_e4m3fn


def test_storage_of_a_cache_in_8_bits():
    reqs = [[KVRequest(2, 64, eight_bit=True)], [KVRequest(2, 64, 32, eight_bit=True)], [KVRequest(2, 64, eight_bit=True)]]
    cache = Cache(reqs, 3, 640, 256, torch.bfloat16, "cpu", F8)
    for u in range(3):
        kv = cache.unit(u).kv
        assert kv.k.dtype == F8 and kv.v.dtype == F8 and kv.k.shape == (11, 2, 64, 64)
        assert kv.k_exp.dtype == torch.int8 and kv.k_exp.shape == (11, 2, 4) == kv.v_exp.shape
        assert kv.k_exp.data_ptr() != kv.v_exp.data_ptr()
    assert cache.unit(0).kv.k_exp.data_ptr() != cache.unit(2).kv.k_exp.data_ptr()
    assert cache.bytes() == 3 * 11 * 2 * (2 * 64 * 64 + 2 * 4)
    plain = Cache(reqs, 3, 640, 256, torch.bfloat16, "cpu")
    assert plain.unit(0).kv.k.dtype == torch.bfloat16 and plain.unit(0).kv.k_exp is None and plain.unit(0).kv.v_exp is None
    assert plain.bytes() == 3 * 11 * 2 * 2 * 64 * 64 * 2


@pytest.mark.parametrize("req", [KVRequest(2, 64), KVRequest(2, 64, v_head_dim=32, eight_bit=True),
                                 KVRequest(1, 64, values_in_keys=48, eight_bit=True),
                                 KVRequest(2, 64, 32, keep_first=4, eight_bit=True)])
def test_mixers_that_do_not_know_it_are_refused(req):
    with pytest.raises(ValueError, match="cannot be held in 8 bits"):
        Cache([[req]], 2, 128, 128, torch.bfloat16, "cpu", F8)
    Cache([[req]], 2, 128, 128, torch.bfloat16, "cpu")


def test_a_position_encoding_that_writes_the_cache_itself_is_asked():
    from llm_infer_engine_b200.parts.attention import GroupedQueryAttention
    from llm_infer_engine_b200.parts.base import PositionEncoding
    from llm_infer_engine_b200.parts.rope import NoEncoding, RotaryEncoding
    layer = GroupedQueryAttention.__new__(GroupedQueryAttention)
    layer.n_kv_heads, layer.head_dim, layer.window = 2, 64, 0
    for position, knows in ((RotaryEncoding, True), (NoEncoding, True), (PositionEncoding, False)):
        layer.position = position
        assert layer.cache_requests() == [KVRequest(2, 64)] and layer.cache_requests()[0].eight_bit is knows


def test_other_types_are_refused():
    with pytest.raises(ValueError, match="held in"):
        Cache([[KVRequest(2, 64, eight_bit=True)]], 2, 128, 128, torch.bfloat16, "cpu", torch.float16)


def test_a_request_is_the_same_whether_or_not_it_may_be_held_in_8_bits():
    assert KVRequest(2, 64) == KVRequest(2, 64, eight_bit=True)
    assert KVRequest(2, 64).geometry() == KVRequest(2, 64, eight_bit=True).geometry()


def test_names():
    bf, f32 = torch.bfloat16, torch.float32
    for name in ("auto", None, "bfloat16", "bf16", bf):
        assert resolve_cache_dtype(name, bf) is bf
    for name in ("float8_e4m3", "float8_e4m3fn", "fp8", F8):
        assert resolve_cache_dtype(name, bf) is F8 and resolve_cache_dtype(name, f32) is F8
    for name, dtype in (("bfloat16", f32), ("float32", bf), ("int8", bf), (torch.float16, bf)):
        with pytest.raises(EngineError, match="cache_dtype"):
            resolve_cache_dtype(name, dtype)


def test_command_line_option(monkeypatch):
    from llm_infer_engine_b200.cli import main as cli
    monkeypatch.delenv("LLM_CACHE_DTYPE", raising=False)
    parser = cli.build_parser()
    assert cli.resolve_all(parser.parse_args([]), {})["cache_dtype"] == "auto"
    assert cli.resolve_all(parser.parse_args(["--cache-dtype", "float8_e4m3"]), {})["cache_dtype"] == "float8_e4m3"
    assert cli.resolve_all(parser.parse_args([]), {"LLM_CACHE_DTYPE": "float8_e4m3"})["cache_dtype"] == "float8_e4m3"
    with pytest.raises(SystemExit):
        parser.parse_args(["--cache-dtype", "int3"])


@pytest.mark.parametrize("call", ["rope_store_fp8", "attention_paged_fp8", "attention_decode_fp8", "attention_decode_fp8_rope",
                                  "attention_prefill_fp8"])
def test_tensors_that_are_not_on_a_gpu_and_heads_that_do_not_divide(call):
    def run(n_q, n_kv, hd=64):
        n = 2
        i32 = torch.zeros(3, dtype=torch.int32)
        table = torch.zeros(3, 2, dtype=torch.int32)
        k = torch.zeros(5, n_kv, 64, hd).to(F8)
        e = torch.zeros(5, n_kv, 4, dtype=torch.int8)
        q, out = torch.zeros(n, n_q * hd, dtype=torch.bfloat16), torch.zeros(n, n_q * hd, dtype=torch.bfloat16)
        qkv = torch.zeros(n, (n_q + 2 * n_kv) * hd, dtype=torch.bfloat16)
        angles = torch.zeros(64, hd // 2, 2)
        if call == "rope_store_fp8":
            ops.rope_store_fp8(qkv, out, k, k, e, e, angles, i32, i32, i32, table, 2, 1, n_q, n_kv, hd, hd)
        elif call == "attention_paged_fp8":
            ops.attention_paged_fp8(q, k, k, e, e, out, i32, i32, i32, table, n_q, n_kv, hd, 0.125)
        elif call == "attention_decode_fp8":
            ops.attention_decode_fp8(q, k, k, e, e, out, i32, i32, table, n_q, n_kv, hd, 0.125)
        elif call == "attention_decode_fp8_rope":
            ops.attention_decode_fp8_rope(qkv, k, k, e, e, out, angles, i32, i32, table, n_q, n_kv, hd, 0.125)
        else:
            ops.attention_prefill_fp8(q, k, k, e, e, out, i32, i32, i32, table, 2, 1, n_q, n_kv, hd, 0.125)

    with pytest.raises(ops.KernelError, match="CUDA tensor"):
        run(4, 2)
    with pytest.raises(ops.KernelError, match="multiple"):
        run(5, 2)
    if call != "rope_store_fp8" and call != "attention_paged_fp8":
        with pytest.raises(ops.KernelError, match="not supported"):
            run(4, 2, 80)


def test_the_plain_exponent_is_the_smallest_that_fits():
    for big, e in ((448.0, 0), (448.1, 1), (447.9, 0), (224.0, -1), (1.0, -8), (0.875, -9), (0.8751, -8), (0.0, -64),
                   (1e-30, -64), (2.0 ** 127, 119), (448.0 * 2.0 ** -64, -64), (float("inf"), -64)):
        assert fp8_cache.exponent_of(torch.tensor([big, -big / 3])) == (fp8_cache.exponent_of(torch.tensor([0.0]))
                                                                       if big == float("inf") else e), big


def test_scratch_is_held_until_the_launch_is_in_the_stream(monkeypatch):
    """Given back before the call, its memory could go to another host thread, or be unmapped, before the kernel is launched."""
    import weakref
    made = []

    def empty(*shape, **kw):
        t = torch.zeros(*shape, **kw)
        made.append(weakref.ref(t))
        return t

    calls = []

    def launch(*args):
        calls.append(args)
        if not args[1]:
            return ops._NEEDS_SCRATCH
        assert made[-1]() is not None and made[-1]().data_ptr() == args[1]
        return 0

    monkeypatch.setattr(ops.torch, "empty", empty)
    monkeypatch.setitem(ops._fp8_scratch_floats, ("some_family", (1, 2)), 64)
    ops._with_scratch("some_call", "some_family", launch, ("before",), ("after",), (1, 2), "cpu")
    assert [c[0] for c in calls] == ["before"] * 2 and [c[2] for c in calls] == ["after"] * 2 and len(made) == 1


def test_a_timer_counts_a_call_that_is_asked_again_with_scratch_once(monkeypatch):
    from llm_infer_engine_b200.kernels import trace
    marks = []

    class Event:
        def __init__(self, **kw):
            pass

        def record(self):
            marks.append(self)

    monkeypatch.setattr(torch.cuda, "Event", Event)
    timer = trace.KernelTimer()
    answers = [ops._NEEDS_SCRATCH, 0, 0]
    monkeypatch.setattr(trace, "timer", timer)

    class Raw:
        argtypes = restype = None

        def __call__(self, call):
            return answers.pop(0)

    class Library:
        llmie_some_call = Raw()

    monkeypatch.setattr(ops.build, "load", lambda family: Library())
    monkeypatch.setattr(ops, "_apply_pdl", lambda family: None)
    monkeypatch.setitem(ops._fp8_scratch_floats, ("some_family", (1, 2)), 64)
    monkeypatch.setattr(ops, "_fn_cache", {})
    f = ops._fn_by_address("some_family", "llmie_some_call", "3P")
    timer.note(100.0, 7.0)
    ops._with_scratch("some_call", "some_family", f, (1,), (2,), (1, 2), "cpu")
    assert [r[0] for r in timer.records] == ["some"] and timer.records[0][4:] == (100.0, 7.0)
    ops._with_scratch("some_call", "some_family", f, (1,), (2,), (1, 2), "cpu")
    assert len(timer.records) == 2 and timer.records[1][4:] == (0.0, 0.0) and not answers


def test_one_token_steps_that_cannot_be_counted_go_to_the_plain_kernel(monkeypatch):
    """The decode kernel counts a step's positions in 32 bits, by items of a KV head, not of a query head; a step beyond that is refused by
    the kernels of its own, and the caller goes on with append and plain attention."""
    from types import SimpleNamespace
    from llm_infer_engine_b200.engine.plan import KernelPlan
    from llm_infer_engine_b200.parts.base import AttentionOptions
    assert ops.attention_decode_fp8_counts(512, 64, 8, 16384) and ops.attention_decode_fp8_counts(512, 64, 4, 16384)
    assert ops.attention_decode_fp8_counts(953, 64, 64, 16384) and not ops.attention_decode_fp8_counts(954, 64, 64, 16384)
    assert not ops.attention_decode_fp8_counts(954, 64 * 8, 64, 16384)
    assert not ops.attention_decode_fp8_counts(954, 64 * 17, 32, 16384)         # two chunks of query heads
    called = []
    monkeypatch.setattr(ops, "attention_decode_fp8", lambda *a: called.append("decode"))
    monkeypatch.setattr(ops, "attention_decode_fp8_rope", lambda *a: called.append("step"))
    plan = KernelPlan(SimpleNamespace(dtype=torch.bfloat16, decode_attention="auto"))
    x = torch.zeros(1, 1, dtype=torch.bfloat16)
    for lanes, pages, taken in ((512, 16384, True), (954, 16384, False)):
        kv = SimpleNamespace(k=None, v=None, k_exp=x, v_exp=x, block_table=torch.empty(1, pages, dtype=torch.int32))
        ctx = SimpleNamespace(decode=True, n_seqs=lanes, seq_slot=None, seq_kvlen=None, max_kv_len=10)
        options = AttentionOptions(scale=0.125)
        assert plan.attention(ctx, x, kv, x, 64, 64, 64, options) is taken
        assert plan.attention_with_rope(ctx, x, x, kv, x, 64, 64, 64, options, True) is taken
        assert called == (["decode", "step"] if taken else [])
        called.clear()
