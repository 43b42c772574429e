"""Decode attention over the 4-bit KV cache, rows in and out, accumulated weights and
rotary positions with three axes, against the float64 restatement (oracle/q4_ref.py).

Held rows are compared exactly: both sides decide the codes in f64, and a value lies
within 2^-52 of a border with a probability of about 1e-12.

Tolerances.  A score is a sum of 256 f32 products; each addition rounds by at most
2^-24 of a partial sum, and |q.k| / 16 <= 16 for normalised rows, so random rounding
gives sqrt(256) * 2^-24 * 16 = 1.5e-5 on a score and the same, relatively, on its
probability.  Outputs are averages of values with those weights: |error| <= 1.5e-5 *
max|v| (OUT_TOL, 2e-5 with the f32 norm and the gate).  Weights are sums of 6
probabilities: relative 2e-5 of each plus 2^-24 per addition to what was there."""
import numpy as np
import pytest

from daiza_b200._ffi import DZ_EINVAL, DZ_ESTATE, DzError
from oracle import q4_ref as R

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

OUT_TOL, W_TOL = 2e-5, 2e-5


def dev(x, dtype=None):
    return torch.tensor(np.ascontiguousarray(x), dtype=dtype or torch.float32, device="cuda")


class Model:
    """A context with one full-attention layer and a float64 cache per sequence beside it."""

    def __init__(self, caps, kvc=4, seed=0, track=False, sections=(11, 11, 10), interleaved=False):
        import daiza_b200 as dz
        self.rng = np.random.default_rng(seed)
        self.kvc, self.nq = kvc, 6 * kvc
        self.ctx = dz.Context(0, dz.default_config(n_layers=1, full_attention_interval=1, kv_heads=(0, kvc)))
        self.qn, self.kn = (1 + 0.1 * self.rng.standard_normal((2, 256))).astype(np.float32)
        self.ctx.set_attn_params(0, self.qn, self.kn)
        self.ctx.set_rope_axes(sections, interleaved)
        self.axis = R.axes(sections, interleaved)
        self.ctx.cache_create_q4(caps, track=track)
        self.refs = [R.Cache(kvc) for _ in caps]

    def normal(self, *shape):
        return self.rng.standard_normal(shape).astype(np.float32)

    def fill(self, seq, n, loud=1.0):
        k, v = self.normal(n, self.kvc, 256), loud * self.normal(n, self.kvc, 256)
        self.ctx.kv_import(0, seq, dev(k), dev(v))
        self.refs[seq] = R.Cache(self.kvc, k, v)

    def inputs(self, B):
        return self.normal(B, self.nq, 512), self.normal(B, self.kvc, 256), self.normal(B, self.kvc, 256)

    def decode(self, ids, inputs=None, pos=None, stream=None):
        qg, k, v = self.inputs(len(ids)) if inputs is None else inputs
        out = torch.full((len(ids), self.nq * 256), -7.0, device="cuda")
        self.ctx.gqa_decode_q4(0, ids, dev(qg), dev(k), dev(v), out, pos=pos)
        want = np.concatenate([self.refs[s].extend(qg[b:b + 1], k[b:b + 1], v[b:b + 1], self.qn, self.kn,
                                                   None if pos is None else np.asarray(pos)[b:b + 1], self.axis)
                               for b, s in enumerate(ids)])
        return out.cpu().numpy().astype(np.float64).reshape(want.shape), want

    def check_decode(self, ids, **kw):
        got, want = self.decode(ids, **kw)
        for b, s in enumerate(ids):
            err = np.abs(got[b] - want[b]).max()
            assert err <= OUT_TOL * np.abs(self.refs[s].v).max(), f"row {b} (seq {s}): {err:.2e}"

    def check_held(self, seq):
        k, v = self.ctx.kv_export(0, seq)
        assert np.array_equal(k, self.refs[seq].k) and np.array_equal(v, self.refs[seq].v), f"seq {seq}"

    def weights(self, ids):
        n = [self.ctx.kv_len(0, s) for s in ids]
        out = torch.empty(self.kvc * sum(n), device="cuda")
        self.ctx.kv_weights_q4(0, ids, out)
        parts = np.split(out.cpu().numpy(), np.cumsum([self.kvc * m for m in n])[:-1])
        return [p.reshape(self.kvc, m) for p, m in zip(parts, n)]

    def check_weights(self, ids):
        for s, w in zip(ids, self.weights(ids)):
            want = self.refs[s].w
            assert np.all(np.abs(w - want) <= W_TOL * np.maximum(want, want.mean())), f"seq {s}"

    def done(self):
        assert self.ctx.device_error() == 0
        self.ctx.close()


# ---- rows in and out ---------------------------------------------------------------------
@pytest.mark.parametrize("n,kvc", [(1, 4), (15, 1), (16, 4), (17, 2), (100, 4), (4099, 1)])
def test_import_and_export(n, kvc):
    m = Model([n, 7], kvc=kvc, seed=n)
    m.fill(0, n)
    m.check_held(0)
    k, v = m.ctx.kv_export(0, 0)
    m.ctx.kv_import(0, 0, k, v)                       # held values hold themselves
    m.check_held(0)
    m.done()


def test_import_of_extremes():
    m = Model([40], seed=3)
    scale = np.float32(10.0) ** np.linspace(-9, 7, 40, dtype=np.float32)[:, None, None]
    k, v = m.normal(40, 4, 256) * scale, m.normal(40, 4, 256) * scale[::-1]
    k[3, 1, 5], k[3, 1, 200], v[4, 0, 31], v[4, 0, 32] = np.nan, np.inf, -np.inf, np.nan
    k[5], v[6] = 0.0, np.nan
    v[7, 2, :32] = np.float32(2.0 ** -17 * 3.5)       # half a grid step of the smallest scales: a tie
    k[8, 0, :8] = [7, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, -7]
    k[8, 0, 8:32] = 0.0
    m.ctx.kv_import(0, 0, k, v)
    m.refs[0] = R.Cache(4, k, v)
    m.check_held(0)
    m.done()


def test_lengths_of_several_sequences():
    m = Model([50, 33, 20], seed=41)
    for s, n in enumerate((50, 0, 20)):
        if n:
            m.fill(s, n)
    assert m.ctx.kv_lens(0, [2, 0, 1, 2]) == [20, 50, 0, 20]
    for bad in ([3], [-1], []):
        refused(DZ_EINVAL, m.ctx.kv_lens, 0, bad)
    refused(DZ_EINVAL, m.ctx.kv_lens, 1, [0])
    m.done()


def test_rows_of_several_sequences():
    m = Model([50, 33, 20], seed=4)
    for s, n in enumerate((50, 33, 20)):
        m.fill(s, n)
    ids, first, count = [2, 0, 1], [3, 17, 33], [17, 33, 0]
    k, v = (torch.full((50, 4, 256), -7.0, device="cuda") for _ in "kv")
    m.ctx.kv_rows_q4(0, ids, first, count, k, v)
    for got, name in ((k, "k"), (v, "v")):
        want = np.concatenate([getattr(m.refs[s], name)[a:a + c] for s, a, c in zip(ids, first, count)])
        assert np.array_equal(got.cpu().numpy(), want)
    m.ctx.kv_rows_q4(0, [0], [0], [0], k[:0], v[:0])   # none at all
    m.done()


# ---- decode ------------------------------------------------------------------------------
@pytest.mark.parametrize("kvc", [1, 4])
@pytest.mark.parametrize("n", [0, 1, 14, 15, 16, 17, 31, 32, 33, 255, 1000, 4111])
def test_decode_lengths(n, kvc):
    m = Model([n + 1], kvc=kvc, seed=10 * n + kvc)
    if n:
        m.fill(0, n)
    m.check_decode([0])
    m.check_held(0)
    m.done()


def test_decode_ragged_batch_in_any_order():
    lens = [0, 700, 16, 2049, 5, 129, 64, 1, 3500, 47]
    m = Model([n + 3 for n in lens], seed=20)
    for s, n in enumerate(lens):
        if n:
            m.fill(s, n)
    for ids in ([7, 3, 0, 9, 1], [8, 2, 4, 6, 5], list(range(10))):
        m.check_decode(ids)
    for s in range(10):
        m.check_held(s)
    m.done()


def test_decode_many_steps_across_tiles_and_truncation():
    m = Model([80, 80], seed=21, track=True)
    m.fill(0, 5)
    for step in range(40):
        m.check_decode([0, 1] if step % 3 else [1, 0])
    m.check_held(0)
    m.check_held(1)
    m.check_weights([0, 1])
    m.ctx.kv_truncate(0, 0, 21)
    r = m.refs[0]
    r.k, r.v, r.w = r.k[:21], r.v[:21], r.w[:, :21]
    for _ in range(20):
        m.check_decode([0])
    m.check_held(0)
    m.check_weights([0])                              # a slot that is taken again starts anew
    m.done()


def test_decode_more_sequences_than_one_launch_takes():
    m = Model([4] * 300, kvc=1, seed=22, track=True)
    ids = [int(i) for i in m.rng.permutation(300)]
    for _ in range(2):
        m.check_decode(ids)
    m.check_weights(ids)
    m.done()


def test_decode_long_context_is_split():
    m = Model([70001], kvc=1, seed=23, track=True)
    m.fill(0, 70000)
    m.check_decode([0])
    m.check_weights([0])
    m.done()


@pytest.mark.parametrize("interleaved,sections", [(False, (11, 11, 10)), (True, (11, 11, 10)), (False, (32, 0, 0)),
                                                  (True, (20, 5, 7)), (False, (0, 0, 32))])
def test_decode_three_axes(interleaved, sections):
    m = Model([60, 60], seed=24, sections=sections, interleaved=interleaved)
    m.fill(0, 20)
    pos = [[20, 25, 31], [1000000, 7, 2 ** 31 - 1]]
    m.check_decode([0, 1], pos=pos)
    m.check_decode([0, 1], pos=[[21, 0, 0], [1000001, 1000001, 1000001]])
    m.check_held(0)
    m.check_held(1)
    m.done()


def test_decode_extreme_inputs():
    """Sharp softmax, large and tiny values, infinities in v: held saturated, and finite."""
    m = Model([40], seed=25)
    m.fill(0, 30, loud=300.0)
    qg, k, v = m.inputs(1)
    m.qn *= 30
    m.ctx.set_attn_params(0, m.qn, m.kn)
    got, want = m.decode([0], inputs=(qg, k, v))
    # scores reach 30 * 16: their rounding, sqrt(256) * 2^-24 * 480, is 4.6e-4
    assert np.abs(got - want).max() <= 5e-4 * np.abs(m.refs[0].v).max()
    v[0, 1, 7], v[0, 2, 9] = np.inf, np.nan
    qg[0, :, 256:] = 200.0 * np.sign(qg[0, :, 256:])  # gates of 0 and 1
    got, want = m.decode([0], inputs=(qg * np.float32(1e-3), k, v * np.float32(1e-4)))
    assert np.all(np.isfinite(got))
    assert np.abs(got - want).max() <= 5e-4 * np.abs(m.refs[0].v).max()
    m.check_held(0)
    m.done()


@pytest.mark.parametrize("size", [1e-30, 1e-20, 1e12, 1e19, 1e30, 3e38])
def test_decode_keys_of_any_size(size):
    """K is normalised in f64: squares below and above f32's range count as they are."""
    m = Model([40], seed=31)
    m.fill(0, 19)
    qg, k, v = m.inputs(1)
    k = np.clip(k, -1, 1) * np.float32(size)
    k[0, 1, 100:] = 0.0
    got, want = m.decode([0], inputs=(qg, k, v))
    assert np.abs(got - want).max() <= OUT_TOL * np.abs(m.refs[0].v).max()
    m.check_held(0)
    m.done()


def test_decode_zero_query_and_equal_keys():
    m = Model([20], seed=26, track=True)
    k = np.repeat(m.normal(1, 4, 256), 17, 0)
    v = m.normal(17, 4, 256)
    m.ctx.kv_import(0, 0, k, v)
    m.refs[0] = R.Cache(4, k, v)
    qg, k1, v1 = m.inputs(1)
    qg[0, :3, :256] = 0.0
    got, want = m.decode([0], inputs=(qg, k1, v1))
    assert np.abs(got - want).max() <= OUT_TOL * np.abs(m.refs[0].v).max()
    m.check_weights([0])
    m.done()


def test_decode_on_another_stream_and_in_a_replayed_graph():
    m = Model([600, 300], seed=27)
    m.fill(0, 500)
    m.fill(1, 200)
    qg, k, v = m.inputs(2)
    out = torch.empty(2, 6144, device="cuda")
    tensors = dev(qg), dev(k), dev(v), out
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    m.ctx.gqa_decode_q4(0, [0, 1], *tensors, stream=side)
    side.synchronize()
    first = out.clone()
    m.ctx.kv_truncate(0, 0, 500)
    m.ctx.kv_truncate(0, 1, 200)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m.ctx.gqa_decode_q4(0, [0, 1], *tensors)
    for _ in range(3):                                # a replay takes the same step again
        out.fill_(-7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, first)
    want = np.concatenate([m.refs[s].extend(qg[s:s + 1], k[s:s + 1], v[s:s + 1], m.qn, m.kn) for s in (0, 1)])
    assert np.abs(first.cpu().numpy().reshape(want.shape) - want).max() <= OUT_TOL * np.abs(m.refs[0].v).max()
    m.check_held(1)
    m.done()


# ---- accumulated weights -----------------------------------------------------------------
def test_weights_set_read_and_accumulate():
    m = Model([40, 50, 10], seed=28, track=True)
    m.fill(0, 20)
    m.fill(1, 37)
    assert not any(w.any() for w in m.weights([1, 0, 2]))
    new = [np.abs(m.normal(4, n)) for n in (37, 20)]
    m.ctx.kv_set_weights_q4(0, [1, 0], dev(np.concatenate([w.ravel() for w in new])))
    m.refs[1].w, m.refs[0].w = (w.astype(np.float64) for w in new)
    m.check_weights([0, 1])
    m.check_decode([1, 2, 0])
    m.check_weights([0, 1, 2])
    m.done()


# ---- the other calls on 4-bit caches -------------------------------------------------------
def test_session_and_snapshot_hold_what_the_cache_holds(tmp_path):
    import daiza_b200 as dz
    ctx = dz.Context(0, dz.default_config(n_layers=4))
    rng = np.random.default_rng(29)
    ctx.cache_create_q4([64, 64])
    k, v = rng.standard_normal((2, 30, 4, 256)).astype(np.float32)
    ctx.kv_import(3, 0, k, v)
    ctx.snapshot_reserve(1)
    ctx.snapshot_save(0, 0)
    ctx.session_save(0, tmp_path / "s.dzss", pos=30)
    held = ctx.kv_export(3, 0)
    assert np.array_equal(held[0], R.hold(k)) and np.array_equal(held[1], R.hold(v))
    ctx.session_load(1, tmp_path / "s.dzss")
    for a, b in zip(held, ctx.kv_export(3, 1)):
        assert np.array_equal(a, b)
    ctx.snapshot_restore(0, 0)
    ctx.kv_truncate(3, 0, 10)
    with pytest.raises(DzError) as e:                 # rows below the saved length may change
        ctx.snapshot_restore(0, 0)
    assert e.value.status == DZ_ESTATE
    ctx.cache_reset(0)
    assert ctx.kv_len(3, 0) == 0
    ctx.close()


# ---- rotary positions of three axes ----------------------------------------------------------
@pytest.mark.parametrize("T,kvc,dtype,interleaved", [(1, 4, "float32", False), (3, 1, "float32", True),
                                                     (300, 4, "float32", True), (1, 2, "bfloat16", True),
                                                     (261, 4, "bfloat16", False)])
def test_qk_mrope(T, kvc, dtype, interleaved):
    """f32: the angle's sine and cosine to 2^-22, two products and the norm (256 squares): 2e-6 of the row's largest
    value.  bf16 adds its rounding, 2^-8 of the value."""
    m = Model([4], kvc=kvc, seed=T, interleaved=interleaved)
    dt = getattr(torch, dtype)
    qg, k = dev(m.normal(T, m.nq, 512), dt), dev(m.normal(T, kvc, 256), dt)
    pos = m.rng.integers(0, 1 << 20, (T, 3))
    pos[0] = [0, 2 ** 31 - 1, 5]
    q_out, k_out = torch.empty(T, m.nq, 256, dtype=dt, device="cuda"), torch.empty_like(k)
    m.ctx.qk_mrope(0, dev(pos, torch.int32), qg, k, q_out, k_out)
    for got, x, norm, c in ((q_out, qg[..., :256], m.qn, 1 / 16), (k_out, k, m.kn, 1.0)):
        want = c * R.turn(x.double().cpu().numpy(), norm, pos, m.axis)
        rounding = 2.0 ** -8 * np.abs(want) if dtype == "bfloat16" else 0.0
        err = np.abs(got.double().cpu().numpy() - want)
        assert np.all(err <= 2e-6 * np.abs(want).max(-1, keepdims=True) + rounding), err.max()
    m.ctx.qk_mrope(0, dev(pos, torch.int32), qg, k, q_out, k)      # k in place
    assert torch.equal(k, k_out)
    m.done()


# ---- refusals ------------------------------------------------------------------------------
def refused(status, call, *a, **kw):
    with pytest.raises(DzError) as e:
        call(*a, **kw)
    assert e.value.status == status, str(e.value)


def test_refusals():
    import daiza_b200 as dz
    m = Model([20, 20], seed=30)
    m.fill(0, 20)
    m.fill(1, 5)
    qg, k, v = (dev(x) for x in m.inputs(2))
    out = torch.empty(2, 6144, device="cuda")
    one = qg[:1], k[:1], v[:1], out[:1]
    c = m.ctx
    refused(DZ_ESTATE, c.gqa_decode_q4, 0, [0], *one)                            # full
    refused(DZ_ESTATE, c.gqa_decode_q4, 0, [1, 0], qg, k, v, out)                # one of two full: nothing happens
    assert c.kv_len(0, 1) == 5
    refused(DZ_EINVAL, c.gqa_decode_q4, 0, [2], *one)
    refused(DZ_EINVAL, c.gqa_decode_q4, 0, [1, 1], qg, k, v, out)
    refused(DZ_EINVAL, c.gqa_decode_q4, 1, [1], *one)
    refused(DZ_EINVAL, c.gqa_decode_q4, 0, [1], *one, pos=[[1, 2, -3]])
    refused(DZ_EINVAL, c.gqa_decode_q4, 0, [1], *one, pos=[[1, 2]])
    refused(DZ_EINVAL, c.gqa_decode_q4, 0, [1], qg, *one[1:])                    # two rows for one sequence
    refused(DZ_EINVAL, c.gqa_decode_q4, 0, [1], one[0].cpu(), *one[1:])
    flat = torch.empty(6144 * 2 + 1, device="cuda")[1:]
    refused(DZ_EINVAL, c.gqa_decode_q4, 0, [1], flat, *one[1:])                  # not 16-byte aligned
    refused(DZ_EINVAL, c.kv_rows_q4, 0, [1], [3], [3], k, v)
    refused(DZ_EINVAL, c.kv_rows_q4, 0, [1], [-1], [2], k, v)
    refused(DZ_EINVAL, c.kv_rows_q4, 0, [1], [0], [1], k, v)                     # room for two rows
    refused(DZ_ESTATE, c.kv_weights_q4, 0, [1], torch.empty(20, device="cuda"))  # not tracked
    refused(DZ_ESTATE, c.kv_set_weights_q4, 0, [1], torch.empty(20, device="cuda"))
    # the f32 calls on a 4-bit cache, and the other way round
    refused(DZ_ESTATE, c.gqa_decode, 0, [1], *one)
    refused(DZ_ESTATE, c.gqa_prefill, 0, 1, *one)
    refused(DZ_ESTATE, c.kv_fill_pattern, 0, 1, 4)
    assert c.lib.dz_gqa_decode_noalloc(c.h, 0, 1, np.zeros(1, np.int32).ctypes.data, *[t.data_ptr() for t in one],
                                       None) == DZ_ESTATE
    refused(DZ_ESTATE, c.kv_import, 0, 0, np.zeros((21, 4, 256), np.float32), np.zeros((21, 4, 256), np.float32))
    for sections, inter in (((11, 11, 11), False), ((-1, 22, 11), False), ((8, 14, 10), True), ((11, 10, 11), True)):
        refused(DZ_EINVAL, c.set_rope_axes, sections, inter)
    m.check_decode([1])                                                          # none of it left a trace
    m.check_held(1)
    m.done()
    f = dz.Context(0, dz.default_config(n_layers=2, full_attention_interval=2))
    f.set_attn_params(1, m.qn, m.kn)
    f.cache_create([8])
    refused(DZ_ESTATE, f.gqa_decode_q4, 1, [0], *one)
    refused(DZ_ESTATE, f.kv_rows_q4, 1, [0], [0], [0], k[:0], v[:0])
    refused(DZ_EINVAL, f.qk_mrope, 0, torch.zeros(1, 3, dtype=torch.int32, device="cuda"), one[0], one[1],
            torch.empty(6144, device="cuda"), torch.empty(1024, device="cuda"))  # a DeltaNet layer
    f.cache_create_q4([8])
    f.cache_create([8])                                                          # and back to f32
    f.gqa_decode(1, [0], *one)
    f.close()
