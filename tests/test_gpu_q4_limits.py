"""What the calls on 4-bit caches take at their limits: values, weights and gates of any size, more prompts than one
group of scratch holds, and scratch that grows."""
import numpy as np
import pytest

from daiza_b200._ffi import DZ_ENOMEM, DzError
from oracle import q4_ref as R
from tests.test_gpu_q4 import OUT_TOL, Model, dev
from tests.test_gpu_q4_prefill import MAX_TOL, check, prompt

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_prompt_gates_of_any_size(dtype):
    """A NaN gate gives NaN, -inf 0, and a nearly closed one sigmoid's own small value.  An eighth of it is a reciprocal
    whose results below 2^-126 are flushed to 0: sigmoids below 2^-123 count as 0."""
    m = Model([40], kvc=1, seed=310)
    q, k, v = m.inputs(30)
    gates = np.array([np.nan, np.inf, -np.inf, 200, -200, -30, -45, -60, -80, 60, 0, -87], np.float32)
    q[:, :, 256:256 + 12], q[:, :, 300:312], q[:, :, 399:411] = gates, gates[::-1], gates
    with np.errstate(over="ignore"):
        (got, want), = prompt(m, [0], [30], dtype, inputs=(q, k, v))
    top = np.abs(m.refs[0].v).max()
    nan = np.isnan(want)
    assert nan.any() and np.array_equal(np.isnan(got), nan)
    g = dev(q, getattr(torch, dtype)).double().cpu().numpy()[..., 256:]
    with np.errstate(over="ignore"):
        open_ = 1 / (1 + np.exp(-g))
    step = 2.0 ** -8 if dtype == "bfloat16" else 0.0
    bound = MAX_TOL * top * open_ + step * np.abs(want) + 2.0 ** -123 * top
    assert np.all((np.abs(got - want) <= bound)[~nan])
    m.done()


@pytest.mark.parametrize("size", [1e-30, 1e12, 1e19, 1e30, 3e38])
def test_queries_of_any_size(size):
    """Rows are normalised whatever their size: squares beyond f32's range count as they are, in decode, prompts and the
    rotary pass."""
    m = Model([60, 60], kvc=2, seed=311)
    m.fill(0, 19)
    qg, k, v = m.inputs(40)
    qg[..., :256] = np.clip(qg[..., :256], -1, 1) * np.float32(size)
    k = np.clip(k, -1, 1) * np.float32(size)
    got, want = m.decode([0], inputs=(qg[:1], k[:1], v[:1]))
    assert np.abs(got - want).max() <= OUT_TOL * np.abs(m.refs[0].v).max()
    for dtype in ("float32", "bfloat16"):
        m.ctx.kv_truncate(0, 1, 0)
        m.refs[1] = R.Cache(2)
        check(m, [1], [40], dtype, inputs=(qg, k, v))
        dt = getattr(torch, dtype)
        tq, tk = dev(qg, dt), dev(k, dt)
        pos = m.rng.integers(0, 1 << 20, (40, 3))
        q_out, k_out = torch.empty(40, m.nq, 256, dtype=dt, device="cuda"), torch.empty_like(tk)
        m.ctx.qk_mrope(0, dev(pos, torch.int32), tq, tk, q_out, k_out)
        for out, x, norm, c in ((q_out, tq[..., :256], m.qn, 1 / 16), (k_out, tk, m.kn, 1.0)):
            want = c * R.turn(x.double().cpu().numpy(), norm, pos, m.axis)
            rounding = 2.0 ** -8 * np.abs(want) if dtype == "bfloat16" else 0.0
            err = np.abs(out.double().cpu().numpy() - want)
            assert np.all(err <= 2e-6 * np.abs(want).max(-1, keepdims=True) + rounding + 1e-30), err.max()
        m.ctx.qk_mrope(0, dev(pos, torch.int32), tq, tk, q_out, tk)    # k in place
        assert torch.equal(tk, k_out)
    m.done()


@pytest.mark.parametrize("T,base", [(1, 4), (100, 0), (150, 333)])
def test_prompt_f32_outputs_keep_their_bits(T, base):
    """Zero queries: every P is the same power of two and outputs are plain means, so nothing but the sums' truncation
    (1 + 483 / 16 additions, 4 * 2^-23 each of a sum that grows: 7.4e-6) and a few f32 roundings stand between."""
    m = Model([base + T], kvc=1, seed=312)
    k, v = m.normal(base, 1, 256), 1 + 0.1 * m.normal(base, 1, 256)
    if base:
        m.ctx.kv_import(0, 0, k, v)
        m.refs[0] = R.Cache(1, k, v)
    q, k, v = m.inputs(T)
    q[..., :256] = 0
    (got, want), = prompt(m, [0], [T], inputs=(q, k, 1 + np.float32(0.1) * v))
    assert np.abs(got - want).max() <= 1e-5 * np.abs(m.refs[0].v).max()
    m.done()


@pytest.mark.parametrize("up", [1e5, 1e4, 1e-2, 1e-4])
def test_prompt_norm_weights_of_any_size(up):
    """Queries large or small, keys the other way round: the same scores, and the same tolerance."""
    m = Model([300], kvc=1, seed=313)
    m.qn *= np.float32(up)
    m.kn /= np.float32(up)
    m.ctx.set_attn_params(0, m.qn, m.kn)
    m.check_decode([0])
    m.check_decode([0])
    check(m, [0], [250])
    m.done()


@pytest.mark.parametrize("weight", [3e6, 1e30, 1e37])
def test_prompt_one_large_norm_weight(weight):
    """A query dim beyond f16 that no key answers."""
    m = Model([300], kvc=1, seed=319)
    m.qn[100], m.kn[100] = weight, 0
    if weight > 1e20:                                # what else there is lies too far below for f16: no score at all
        m.qn[:100] = m.qn[101:] = 0
    m.ctx.set_attn_params(0, m.qn, m.kn)
    m.check_decode([0])
    check(m, [0], [250])
    m.done()


def test_prompt_groups_of_sequences():
    """Five sequences of 120000 cached rows: the f16 rows of four fill the scratch of one group."""
    n, lens = 120000, [3, 1, 40, 2, 130]
    m = Model([n + t for t in lens], kvc=4, seed=314)
    torch.manual_seed(314)
    for s in range(5):
        m.ctx.kv_import(0, s, torch.randn(n, 4, 256, device="cuda"), torch.randn(n, 4, 256, device="cuda"))
    qg, k, v = (dev(x) for x in m.inputs(sum(lens)))
    pos = torch.randint(0, 1 << 20, (sum(lens), 3), device="cuda", dtype=torch.int32)
    out = torch.empty(sum(lens), m.nq * 256, device="cuda")
    m.ctx.gqa_prefill_q4(0, range(5), lens, qg, k, v, out, pos=pos)
    a = 0
    for s, t in enumerate(lens):                      # one at a time: the same bits
        m.ctx.kv_truncate(0, s, n)
        one = torch.empty(t, m.nq * 256, device="cuda")
        b = slice(a, a + t)
        m.ctx.gqa_prefill_q4(0, [s], [t], qg[b], k[b], v[b], one, pos=pos[b])
        assert torch.equal(one, out[b]), s
        a += t
    m.done()


def test_prompt_that_finds_no_memory_leaves_every_length():
    """The second sequence's scratch (2.6 GB) is more than what is left: none of the prompts is appended."""
    n = 640000
    m = Model([100, n + 8], kvc=4, seed=315)
    zeros = torch.zeros(n, 4, 256, device="cuda")
    m.ctx.kv_import(0, 1, zeros, zeros)
    del zeros
    torch.cuda.empty_cache()
    qg, k, v = (dev(x) for x in m.inputs(24))
    out = torch.empty(24, m.nq * 256, device="cuda")
    torch.cuda.synchronize()
    rest = torch.empty(torch.cuda.mem_get_info()[0] - (1 << 30), dtype=torch.uint8, device="cuda")
    with pytest.raises(DzError) as e:
        m.ctx.gqa_prefill_q4(0, [0, 1], [16, 8], qg, k, v, out)
    assert e.value.status == DZ_ENOMEM
    lens = m.ctx.kv_lens(0, [0, 1])
    del rest
    torch.cuda.empty_cache()
    assert lens == [0, n]
    m.ctx.gqa_prefill_q4(0, [0, 1], [16, 8], qg, k, v, out)
    assert m.ctx.kv_lens(0, [0, 1]) == [16, n + 8]
    m.done()


def test_scratch_grows_within_a_capture():
    """The first prompts and evictions of a context may be captured ones: replays give what the plain calls give."""
    m = Model([600] * 4, kvc=1, seed=316, track=True)
    tensors = [dev(x) for x in m.inputs(500)]
    outs = torch.zeros(2, 500, m.nq * 256, device="cuda")
    weights = torch.rand(500, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    kept = torch.zeros(2, 400, dtype=torch.int32, device="cuda")
    prompt_graph, evict_graph = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(prompt_graph):
        m.ctx.gqa_prefill_q4(0, [0], [500], *tensors, outs[0])
    with torch.cuda.graph(evict_graph):
        m.ctx.kv_evict_q4(0, [0], [400], [30], kept=kept[0], into=[2])
    prompt_graph.replay()
    m.ctx.kv_set_weights_q4(0, [0], weights)
    evict_graph.replay()
    m.ctx.gqa_prefill_q4(0, [1], [500], *tensors, outs[1])
    m.ctx.kv_set_weights_q4(0, [1], weights)
    m.ctx.kv_evict_q4(0, [1], [400], [30], kept=kept[1], into=[3])
    torch.cuda.synchronize()
    assert torch.equal(*outs) and torch.equal(*kept)
    for a, b in ((0, 1), (2, 3)):
        assert all(np.array_equal(x, y) for x, y in zip(m.ctx.kv_export(0, a), m.ctx.kv_export(0, b)))
    m.done()


@pytest.mark.parametrize("first", ["prompt", "evict"])
def test_first_call_of_a_context_is_captured(first):
    m = Model([600, 600], kvc=1, seed=318, track=True)
    graph = torch.cuda.CUDAGraph()
    if first == "prompt":
        tensors, out = [dev(x) for x in m.inputs(40)], torch.zeros(2, 40, m.nq * 256, device="cuda")
        with torch.cuda.graph(graph):
            m.ctx.gqa_prefill_q4(0, [0], [40], *tensors, out[0])
        graph.replay()
        m.ctx.gqa_prefill_q4(0, [1], [40], *tensors, out[1])
        torch.cuda.synchronize()
        assert torch.equal(*out)
    else:
        kept = torch.full((1,), -7, dtype=torch.int32, device="cuda")
        m.ctx.gqa_decode_q4(0, [0], *[dev(x) for x in m.inputs(1)], torch.empty(1, m.nq * 256, device="cuda"))
        with torch.cuda.graph(graph):
            m.ctx.kv_evict_q4(0, [0], [1], [0], kept=kept)
        graph.replay()
        torch.cuda.synchronize()
        assert kept.item() == 0
    m.done()


def test_scratch_goes_with_the_caches():
    """The prompt behind 20000 rows takes 80 MB of scratch; smaller caches in the same context give it back."""
    m = Model([20000], kvc=4, seed=317)
    zeros = torch.zeros(20000 - 8, 4, 256, device="cuda")
    m.ctx.kv_import(0, 0, zeros, zeros)
    qg, k, v = (dev(x) for x in m.inputs(8))
    m.ctx.gqa_prefill_q4(0, [0], [8], qg, k, v, torch.empty(8, m.nq * 256, device="cuda"))
    m.ctx.cache_create_q4([16])
    torch.cuda.synchronize()
    small = torch.cuda.mem_get_info()[0]
    m.ctx.cache_create_q4([16])
    m.ctx.close()
    torch.cuda.synchronize()
    assert torch.cuda.mem_get_info()[0] - small <= 32 << 20


def test_rows_and_weights_of_more_sequences_than_one_launch_takes():
    n = [1 + s % 19 for s in range(300)]
    m = Model(n, kvc=2, seed=320, track=True)
    for s in range(300):
        m.fill(s, n[s])
    ids = [int(i) for i in m.rng.permutation(300)]
    first, count = [n[s] // 3 for s in ids], [n[s] - n[s] // 3 for s in ids]
    k, v = (torch.full((sum(count), 2, 256), -7.0, device="cuda") for _ in "kv")
    m.ctx.kv_rows_q4(0, ids, first, count, k, v)
    for got, name in ((k, "k"), (v, "v")):
        assert np.array_equal(got.cpu().numpy(), np.concatenate([getattr(m.refs[s], name)[a:] for s, a in zip(ids, first)]))
    new = [np.abs(m.normal(2, n[s])) for s in ids]
    m.ctx.kv_set_weights_q4(0, ids, dev(np.concatenate([w.ravel() for w in new])))
    for w, got in zip(new, m.weights(ids)):
        assert np.array_equal(w, got)
    m.done()


def test_positions_of_more_prompts_than_one_launch_takes():
    lens = [s % 4 for s in range(300)]
    m = Model([8] * 300, kvc=1, seed=321, interleaved=True)
    pos = m.rng.integers(0, 1 << 20, (sum(lens), 3))
    check(m, list(range(299, -1, -1)), lens[::-1], pos=pos)
    m.check_decode(list(range(300)), pos=[[7, 8, s] for s in range(300)])
    m.done()
