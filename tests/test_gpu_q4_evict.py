"""Eviction from 4-bit KV caches by accumulated attention weight (dz_kv_evict_q4) against
the float64 restatement: indices, held rows and weights are compared exactly, since
nothing is computed on the way."""
import numpy as np
import pytest

from daiza_b200._ffi import DZ_EINVAL, DZ_ESTATE
from oracle import q4_ref as R
from tests.test_gpu_q4 import Model, dev, refused

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def weigh(m, seq, w):
    w = np.asarray(w, np.float32)
    m.ctx.kv_set_weights_q4(0, [seq], dev(w))
    m.refs[seq].w = w.astype(np.float64)


def heavy_tailed(m, n):
    return (np.exp(2 * m.normal(m.kvc, n)) * (m.rng.random((m.kvc, n)) > 0.1)).astype(np.float32)


def evict(m, ids, keep, recent, into=None, **kw):
    """The call on both sides; the restatement's sources stay when it goes elsewhere."""
    import copy
    lens = [min(k, m.ctx.kv_len(0, s)) for k, s in zip(keep, ids)]
    kept = torch.full((m.kvc * sum(lens),), -7, dtype=torch.int32, device="cuda")
    m.ctx.kv_evict_q4(0, ids, keep, recent, kept=kept, into=into, **kw)
    want = []
    for b, s in enumerate(ids):
        to = s if into is None else into[b]
        ref = copy.copy(m.refs[s])
        want.append(ref.evict(keep[b], recent[b]).ravel())
        m.refs[to] = ref
    assert np.array_equal(kept.cpu().numpy(), np.concatenate(want))
    for b, s in enumerate(ids):
        check(m, s if into is None else into[b])
        check(m, s)


def check(m, seq):
    assert m.ctx.kv_len(0, seq) == len(m.refs[seq].k)
    m.check_held(seq)
    assert np.array_equal(m.weights([seq])[0], m.refs[seq].w.astype(np.float32))


@pytest.mark.parametrize("where", ["in place", "elsewhere"])
@pytest.mark.parametrize("n,keep,recent,kvc", [(1, 1, 0, 4), (2, 1, 0, 1), (2, 1, 1, 1), (17, 16, 1, 2), (33, 15, 0, 4),
                                               (100, 99, 50, 1), (100, 1, 0, 4), (100, 100, 3, 1), (100, 500, 400, 2),
                                               (257, 64, 64, 1), (1000, 333, 17, 4), (2049, 2048, 256, 1),
                                               (5000, 4100, 7, 1), (20011, 9000, 128, 2)])
def test_evict(n, keep, recent, kvc, where):
    m = Model([n, min(n, keep)], kvc=kvc, seed=200 + n, track=True)
    m.fill(0, n)
    weigh(m, 0, heavy_tailed(m, n))
    evict(m, [0], [keep], [recent], into=None if where == "in place" else [1])
    m.done()


@pytest.mark.parametrize("kind", ["equal", "zero", "two values", "rising", "falling", "not numbers", "negative"])
def test_evict_ties_and_orders(kind):
    n = 3000
    m = Model([n], kvc=1, seed=210, track=True)
    m.fill(0, n)
    j = np.arange(n, dtype=np.float32)
    w = {"equal": np.full(n, 0.25), "zero": np.zeros(n), "two values": 1 + (j % 7 == 3), "rising": j, "falling": n - j,
         "not numbers": np.where(j % 5 == 0, np.nan, np.where(j % 5 == 1, np.inf, j)),
         "negative": np.where(j % 2 == 0, -j, np.where(j % 3 == 0, -0.0, 0.0))}[kind].astype(np.float32)[None]
    m.ctx.kv_set_weights_q4(0, [0], dev(w))
    m.refs[0].w = np.where(np.isnan(w), -np.inf, w).astype(np.float64)
    keep, recent = 1111, 10
    kept = torch.empty(keep, dtype=torch.int32, device="cuda")
    m.ctx.kv_evict_q4(0, [0], [keep], [recent], kept=kept)
    idx = m.refs[0].evict(keep, recent)
    assert np.array_equal(kept.cpu().numpy(), idx[0])
    m.check_held(0)
    assert np.array_equal(m.weights([0])[0], w[:, idx[0]], equal_nan=True)
    m.done()


def test_evict_a_ragged_batch():
    lens = [500, 1, 47, 3333, 16, 800]
    m = Model(lens + [400] * 6, kvc=2, seed=211, track=True)
    for s, n in enumerate(lens):
        m.fill(s, n)
        weigh(m, s, heavy_tailed(m, n))
    evict(m, [3, 1, 5], [300, 5, 64], [10, 2, 64], into=[8, 1, 6])
    evict(m, [4, 0, 2], [7, 450, 47], [0, 100, 47])
    evict(m, [8, 3], [100, 2000], [0, 2000])
    m.done()


def test_evict_more_sequences_than_one_launch_takes():
    m = Model([20] * 300, kvc=1, seed=212, track=True)
    for s in range(300):
        m.fill(s, 5 + s % 15)
        weigh(m, s, heavy_tailed(m, 5 + s % 15))
    ids = [int(i) for i in m.rng.permutation(300)]
    evict(m, ids, [1 + i % 9 for i in ids], [i % 2 for i in ids])
    m.done()


def test_serving_on_a_budget():
    """A prompt, then decoding with the cache cut to its budget whenever it is full, at the tokens' true positions;
    weights accumulate on the entries that stayed."""
    m = Model([96, 96], kvc=2, seed=213, track=True)
    out = torch.empty(80 + 50, m.nq * 256, device="cuda")
    qg, k, v = m.inputs(130)
    m.ctx.gqa_prefill_q4(0, [0, 1], [80, 50], dev(qg), dev(k), dev(v), out)
    for s, a, n in ((0, 0, 80), (1, 80, 50)):
        m.refs[s].extend(qg[a:a + n], k[a:a + n], v[a:a + n], m.qn, m.kn)
        m.refs[s].w[:] = 0                            # prompts add no weights
    at = [80, 50]
    for step in range(40):
        m.check_decode([0, 1], pos=[[p] * 3 for p in at])
        at = [p + 1 for p in at]
        full = [s for s in (0, 1) if m.ctx.kv_len(0, s) >= 90]
        if full:
            m.check_weights(full)
            got = {s: m.weights([s])[0] for s in full}
            for s in full:                            # the same weights on both sides: near ties fall alike
                m.refs[s].w = got[s].astype(np.float64)
            evict(m, full, [64] * len(full), [16] * len(full))
    assert m.ctx.kv_len(0, 0) < 96 and at == [120, 90]
    m.done()


def test_offsets_beyond_32_bits():
    """The last kv head of a sequence of 6 million slots lies 4.9 GB behind the first: prompt, decode, rows, weights
    and eviction there, and in the sequence behind it."""
    m = Model([6_000_000, 200], kvc=4, seed=218, track=True)
    qg, k, v = m.inputs(130)
    out = torch.empty(130, m.nq * 256, device="cuda")
    m.ctx.gqa_prefill_q4(0, [1, 0], [50, 80], dev(qg), dev(k), dev(v), out)
    for s, a, n in ((1, 0, 50), (0, 50, 80)):
        want = m.refs[s].extend(qg[a:a + n], k[a:a + n], v[a:a + n], m.qn, m.kn)
        got = out[a:a + n].cpu().numpy().reshape(want.shape)
        assert np.abs(got - want).max() <= 2.2e-3 * np.abs(m.refs[s].v).max()
        m.refs[s].w[:] = 0
        m.check_held(s)
    m.check_decode([0, 1])
    m.check_weights([0, 1])
    for s in (0, 1):
        weigh(m, s, heavy_tailed(m, m.ctx.kv_len(0, s)))
    evict(m, [0, 1], [33, 20], [5, 0])
    m.done()


def test_many_long_sequences_at_once():
    """More pairs than clusters of four CTAs fit the GPU, each with more entries than a CTA keeps in registers."""
    n = 9000
    m = Model([n] * 80, kvc=1, seed=219, track=True)
    k, v = m.normal(n, 1, 256), m.normal(n, 1, 256)
    w = heavy_tailed(m, n)
    for s in range(80):
        m.ctx.kv_import(0, s, dev(k), dev(v))
    m.ctx.kv_set_weights_q4(0, list(range(80)), dev(np.concatenate([np.roll(w.ravel(), s) for s in range(80)])))
    keep, recent = 1500, 100
    kept = torch.empty(80 * keep, dtype=torch.int32, device="cuda")
    m.ctx.kv_evict_q4(0, list(range(80)), [keep] * 80, [recent] * 80, kept=kept)
    for s in range(80):
        m.refs[0] = R.Cache(1, k, v)
        m.refs[0].w = np.roll(w.ravel(), s)[None].astype(np.float64)
        idx = m.refs[0].evict(keep, recent)
        assert np.array_equal(kept[s * keep:(s + 1) * keep].cpu().numpy(), idx[0]), f"seq {s}"
        if s % 27 == 0:
            got = m.ctx.kv_export(0, s)
            assert np.array_equal(got[0], m.refs[0].k) and np.array_equal(got[1], m.refs[0].v)
    m.done()


def test_evict_on_another_stream_and_in_a_graph():
    m = Model([900, 300], kvc=4, seed=214, track=True)
    m.fill(0, 900)
    weigh(m, 0, heavy_tailed(m, 900))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    evict(m, [0], [300], [20], into=[1], stream=side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m.ctx.kv_evict_q4(0, [0], [300], [20], into=[1])
    m.ctx.kv_import(0, 1, np.zeros((300, 4, 256), np.float32), np.zeros((300, 4, 256), np.float32))
    graph.replay()
    torch.cuda.synchronize()
    check(m, 1)
    m.done()


def test_snapshots_of_a_rewritten_sequence_are_refused():
    m = Model([50, 50], kvc=1, seed=215, track=True)
    for s in (0, 1):
        m.fill(s, 40)
        weigh(m, s, heavy_tailed(m, 40))
    m.ctx.snapshot_reserve(2)
    m.ctx.snapshot_save(0, 0)
    m.ctx.snapshot_save(1, 1)
    evict(m, [0], [60], [5])                          # nothing leaves
    m.ctx.snapshot_restore(0, 0)
    evict(m, [0], [30], [5], into=[1])
    m.ctx.snapshot_restore(0, 0)
    refused(DZ_ESTATE, m.ctx.snapshot_restore, 1, 1)
    evict(m, [0], [20], [0])
    refused(DZ_ESTATE, m.ctx.snapshot_restore, 0, 0)
    m.done()


def test_refusals():
    m = Model([50, 50, 10], kvc=1, seed=216, track=True)
    m.fill(0, 40)
    m.fill(1, 30)
    c = m.ctx
    refused(DZ_EINVAL, c.kv_evict_q4, 0, [0], [0], [0])
    refused(DZ_EINVAL, c.kv_evict_q4, 0, [0], [10], [11])
    refused(DZ_EINVAL, c.kv_evict_q4, 0, [0], [10], [-1])
    refused(DZ_EINVAL, c.kv_evict_q4, 0, [0, 0], [10, 10], [1, 1])
    refused(DZ_EINVAL, c.kv_evict_q4, 0, [0, 1], [10, 10], [1, 1], into=[2, 2])
    refused(DZ_EINVAL, c.kv_evict_q4, 0, [0, 1], [10, 10], [1, 1], into=[1, 0])   # would overwrite a source
    refused(DZ_EINVAL, c.kv_evict_q4, 0, [0], [10], [1], into=[3])
    refused(DZ_EINVAL, c.kv_evict_q4, 0, [0], [10], [1], into=[1, 2])
    refused(DZ_ESTATE, c.kv_evict_q4, 0, [0], [11], [1], into=[2])                # 11 rows, capacity 10
    refused(DZ_EINVAL, c.kv_evict_q4, 0, [0], [10], [1], kept=torch.empty(9, dtype=torch.int32, device="cuda"))
    refused(DZ_EINVAL, c.kv_evict_q4, 0, [0], [10], [1], kept=torch.empty(10, device="cuda"))
    check(m, 0)
    evict(m, [2, 0], [3, 10], [1, 0])                 # an empty sequence stays empty
    m.done()
    plain = Model([20], kvc=1, seed=217)
    plain.fill(0, 20)
    refused(DZ_ESTATE, plain.ctx.kv_evict_q4, 0, [0], [10], [1])                  # no weights
    plain.done()
