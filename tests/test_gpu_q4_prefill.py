"""Prompts into 4-bit KV caches (dz_gqa_prefill_q4, f32 and bf16) against the float64
restatement; held rows exactly.

Tolerances.  Q and P are rounded to f16 (at most 2^-11, 2^-12.3 rms of a value); for
normalised rows of 256 independent values the score's error is the rms of its 256
products' errors, 2^-12.3 * |q||k| / 16 / 16 = 2e-4 rms, and acts like a relative error of
the probability, P's own rounding adds as much.  The output is a sum of values with
independently perturbed weights: 2-norm error sqrt(2) * 2e-4 = 2.8e-4 of the output's,
held to 6e-4.  Single elements: 4 sigma of the score (8e-4), the same in the
denominator, and 2^-11 of P: 2.2e-3 * max|v|.  bf16 output adds half a step, 2^-8 of the
value (2-norm 2^-8 / sqrt(3))."""
import numpy as np
import pytest

from daiza_b200._ffi import DZ_EINVAL, DZ_ESTATE
from oracle import q4_ref as R
from tests.test_gpu_q4 import OUT_TOL, Model, dev, refused

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

NORM_TOL, MAX_TOL = 6e-4, 2.2e-3


def prompt(m, ids, lens, dtype="float32", pos=None, inputs=None):
    """Runs the call and the restatement; (got, want) per sequence."""
    T, dt = sum(lens), getattr(torch, dtype)
    if inputs is None:
        inputs = m.inputs(T)
    tensors = [dev(x, dt) for x in inputs]
    qg, k, v = (x.float().cpu().numpy() for x in tensors)
    out = torch.full((T, m.nq * 256), -7.0, device="cuda", dtype=dt)
    m.ctx.gqa_prefill_q4(0, ids, lens, *tensors, out, pos=None if pos is None else dev(pos, torch.int32))
    got, pairs, a = out.double().cpu().numpy().reshape(T, m.nq, 256), [], 0
    for s, n in zip(ids, lens):
        w = m.refs[s].w
        want = m.refs[s].extend(qg[a:a + n], k[a:a + n], v[a:a + n], m.qn, m.kn, None if pos is None else pos[a:a + n],
                                m.axis)
        m.refs[s].w = np.pad(w, ((0, 0), (0, n)))     # prompts add no weights
        pairs.append((got[a:a + n], want))
        a += n
    return pairs


def check(m, ids, lens, dtype="float32", **kw):
    step = 2.0 ** -8 if dtype == "bfloat16" else 0.0
    for s, (got, want) in zip(ids, prompt(m, ids, lens, dtype, **kw)):
        if not got.size:
            continue
        top = np.abs(m.refs[s].v).max()
        assert np.all(np.abs(got - want) <= MAX_TOL * top + step * np.abs(want)), f"seq {s}"
        rel = np.linalg.norm(got - want) / np.linalg.norm(want)
        assert rel <= NORM_TOL + step / 3 ** 0.5, f"seq {s}: {rel:.2e}"
        m.check_held(s)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("T,base,kvc", [(1, 0, 4), (2, 13, 1), (15, 0, 1), (16, 0, 4), (17, 15, 2), (127, 1, 1),
                                        (128, 0, 1), (129, 127, 1), (140, 300, 1), (513, 0, 1)])
def test_prompt_lengths(T, base, kvc, dtype):
    m = Model([base + T], kvc=kvc, seed=100 + T + base)
    if base:
        m.fill(0, base)
    check(m, [0], [T], dtype)
    m.done()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_packed_prompts_of_different_lengths(dtype):
    lens = [5, 130, 0, 1, 260, 16, 33]
    bases = [0, 7, 40, 129, 0, 16, 127]
    m = Model([a + b for a, b in zip(lens, bases)], kvc=1, seed=110)
    for s, b in enumerate(bases):
        if b:
            m.fill(s, b)
    order = [3, 0, 6, 2, 4, 1, 5]
    check(m, order, [lens[s] for s in order], dtype)
    assert [m.ctx.kv_len(0, s) for s in range(7)] == [a + b for a, b in zip(lens, bases)]
    m.done()


def test_many_short_prompts():
    m = Model([3] * 300, kvc=1, seed=111)
    ids = [int(i) for i in m.rng.permutation(300)]
    check(m, ids, [1 + i % 3 for i in range(300)])
    m.done()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_more_query_tiles_than_fit_the_gpu_at_once(dtype):
    """Several tiles per cluster, of one and of many key blocks."""
    rng = np.random.default_rng(121)
    lens = [int(n) for n in rng.integers(1, 300, 40)]
    bases = [int(n) for n in rng.integers(0, 2, 40) * rng.integers(1, 500, 40)]
    m = Model([a + b for a, b in zip(lens, bases)], seed=121)
    for s, b in enumerate(bases):
        if b:
            m.fill(s, b)
    check(m, list(range(40)), lens, dtype)
    m.done()


def test_prompt_then_decode_then_prompt():
    m = Model([400, 200], seed=112, track=True)
    check(m, [0, 1], [150, 37])
    for _ in range(3):
        m.check_decode([1, 0])
    check(m, [1], [65], "bfloat16")
    m.check_decode([0, 1])
    m.check_weights([0, 1])
    m.done()


def test_prompt_equals_decode_steps():
    """The same tokens one by one and as a prompt: the same held rows, outputs within the prompt's rounding."""
    m = Model([60, 60], seed=113)
    m.fill(0, 20)
    held = m.ctx.kv_export(0, 0)
    m.ctx.kv_import(0, 1, *held)
    qg, k, v = m.inputs(40)
    out = torch.empty(40, 6144, device="cuda")
    m.ctx.gqa_prefill_q4(0, [0], [40], dev(qg), dev(k), dev(v), out)
    steps = torch.empty(40, 6144, device="cuda")
    for t in range(40):
        m.ctx.gqa_decode_q4(0, [1], dev(qg[t]), dev(k[t]), dev(v[t]), steps[t])
    for a, b in zip(m.ctx.kv_export(0, 0), m.ctx.kv_export(0, 1)):
        assert np.array_equal(a, b)
    top = np.abs(m.ctx.kv_export(0, 0)[1]).max()
    assert (out - steps).abs().max().item() <= (MAX_TOL + OUT_TOL) * top
    m.done()


@pytest.mark.parametrize("interleaved", [False, True])
def test_prompt_positions_of_images(interleaved):
    m = Model([200, 100], kvc=2, seed=114, interleaved=interleaved)
    m.fill(1, 9)
    t = np.arange(150)
    image = (t >= 30) & (t < 94)
    pos = np.stack([np.where(image, 30, t), np.where(image, 30 + (t - 30) // 8, t), np.where(image, 30 + t % 8, t)], 1)
    pos[140:] = [[2 ** 31 - 1, 5, 1 << 20]]
    check(m, [0, 1], [100, 50], pos=pos)
    m.done()


def test_prompt_extremes_stay_in_their_rows():
    """NaN in one sequence's queries, infinities in another's values: neighbours and later keys are not touched."""
    m = Model([200, 200, 200], kvc=1, seed=115)
    qg, k, v = m.inputs(200 + 70 + 90)
    qg[200, 2, :256] = np.nan                         # sequence 1's first token, head 2
    v[275, 0, 3], v[276, 0, 4] = np.inf, np.nan       # sequence 2's values, held saturated and as 0
    k[280, 0, 7] = np.nan                             # its norm is NaN: the row is held as zeros
    out = torch.empty(360, 6 * 256, device="cuda")
    m.ctx.gqa_prefill_q4(0, [0, 1, 2], [200, 70, 90], dev(qg), dev(k), dev(v), out)
    got = out.cpu().numpy().reshape(360, 6, 256)
    bad = ~np.isfinite(got)
    assert bad[200, 2].all()
    bad[200, 2] = False
    assert not bad.any()
    a = 0
    for s, n in enumerate((200, 70, 90)):
        with np.errstate(invalid="ignore"):
            want = m.refs[s].extend(qg[a:a + n], k[a:a + n], v[a:a + n], m.qn, m.kn)
        m.check_held(s)
        ok = np.isfinite(want)
        assert np.abs(np.where(ok, got[a:a + n] - want, 0)).max() <= MAX_TOL * np.abs(m.refs[s].v).max()
        a += n
    m.done()


@pytest.mark.parametrize("loud", [1e-4, 2000.0])
def test_prompt_values_near_the_ends_of_the_scales(loud):
    """Values on the smallest scales' grid, and held near 7 * 896: the outputs keep their bits on the way out."""
    m = Model([500], kvc=1, seed=122)
    m.fill(0, 200, loud=loud)
    q, k, v = m.inputs(300)
    check(m, [0], [300], inputs=(q, k, np.float32(loud) * v))
    m.done()


def test_prompt_query_tile_split():
    """Two contexts that share a kv head's query tiles (qtile_split): together they give the whole, each holds all
    rows; the other's output rows are left as they were."""
    import daiza_b200 as dz
    m = Model([400, 300], kvc=1, seed=116)
    qg, k, v = m.inputs(650)
    whole = torch.empty(650, 6 * 256, device="cuda")
    m.ctx.gqa_prefill_q4(0, [0, 1], [385, 265], dev(qg), dev(k), dev(v), whole)
    out = torch.full_like(whole, -7.0)
    for i in range(2):
        c = dz.Context(0, dz.default_config(n_layers=1, full_attention_interval=1, kv_heads=(0, 1), qtile_split=(i, 2)))
        c.set_attn_params(0, m.qn, m.kn)
        c.cache_create_q4([400, 300])
        c.gqa_prefill_q4(0, [0, 1], [385, 265], dev(qg), dev(k), dev(v), out)
        for s in (0, 1):
            assert np.array_equal(c.kv_export(0, s)[0], m.ctx.kv_export(0, s)[0])
        if i == 0:
            left = out.reshape(650, -1)[:, 0] == -7.0
            assert left[128:256].all() and not left[:128].any() and left[385 + 128:385 + 256].all()
        c.close()
    assert torch.equal(out, whole)
    m.done()


def test_prompt_on_another_stream_and_in_graphs():
    m = Model([300, 300], kvc=1, seed=117)
    a, b = [dev(x) for x in m.inputs(200)], [dev(x) for x in m.inputs(50)]
    oa, ob = (torch.empty(n, 6 * 256, device="cuda") for n in (200, 50))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    m.ctx.gqa_prefill_q4(0, [0], [50], *b, ob, stream=side)
    m.ctx.gqa_prefill_q4(0, [1], [200], *a, oa, stream=side)       # the scratch grows
    side.synchronize()
    first = oa.clone(), ob.clone()
    m.ctx.kv_truncate(0, 0, 0)
    m.ctx.kv_truncate(0, 1, 0)
    graphs = [torch.cuda.CUDAGraph() for _ in "ab"]
    with torch.cuda.graph(graphs[0]):
        m.ctx.gqa_prefill_q4(0, [1], [200], *a, oa)
    with torch.cuda.graph(graphs[1]):
        m.ctx.gqa_prefill_q4(0, [0], [50], *b, ob)
    m.ctx.kv_truncate(0, 0, 0)
    big = [dev(x) for x in m.inputs(290)]                          # outgrows the scratch that the graphs hold
    m.ctx.gqa_prefill_q4(0, [0], [290], *big, torch.empty(290, 6 * 256, device="cuda"))
    for i in (0, 1, 0):
        (oa, ob)[i].fill_(-7.0)
        graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal((oa, ob)[i], first[i])
    m.done()


def test_scratch_of_growing_prompts_stays_bounded():
    """Scratch that was outgrown stays (captured graphs may hold it): all of it together below the last one's size."""
    m = Model([1300], kvc=4, seed=119)
    tensors = [dev(x) for x in m.inputs(1300)]
    out = torch.empty(1300, 24 * 256, device="cuda")
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    for T in range(20, 1301, 16):
        m.ctx.kv_truncate(0, 0, 0)
        m.ctx.gqa_prefill_q4(0, [0], [T], *(x[:T] for x in tensors), out[:T])
    torch.cuda.synchronize()
    need = 1300 * 24 * 512 + 1408 * 4 * 1024
    assert free - torch.cuda.mem_get_info()[0] <= 4 * need + (64 << 20)
    m.done()


def test_two_contexts_at_once():
    """Contexts share nothing: calls of two of them overlap on two streams."""
    ms = [Model([700], kvc=1, seed=120 + i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in ms]
    work = []
    for m in ms:
        t, u = m.inputs(600), m.inputs(1)
        work.append((t, [dev(x) for x in t], u, [dev(x) for x in u], torch.empty(600, 1536, device="cuda"),
                     torch.empty(1, 1536, device="cuda")))
    torch.cuda.synchronize()
    for m, st, (_, t, _, u, o, o1) in zip(ms, streams, work):
        m.ctx.gqa_prefill_q4(0, [0], [600], *t, o, stream=st)
        m.ctx.gqa_decode_q4(0, [0], *u, o1, stream=st)
    torch.cuda.synchronize()
    for m, (t, _, u, _, o, o1) in zip(ms, work):
        for x, got, tol in ((t, o, MAX_TOL), (u, o1, OUT_TOL)):
            want = m.refs[0].extend(*x, m.qn, m.kn)
            got = got.cpu().numpy().reshape(want.shape)
            assert np.abs(got - want).max() <= tol * np.abs(m.refs[0].v).max()
        m.check_held(0)
        m.done()


def test_refusals():
    m = Model([20, 20], kvc=1, seed=118)
    m.fill(0, 15)
    q, k, v = (dev(x) for x in m.inputs(6))
    out = torch.empty(6, 6 * 256, device="cuda")
    c = m.ctx
    refused(DZ_ESTATE, c.gqa_prefill_q4, 0, [0], [6], q, k, v, out)              # 15 + 6 > 20
    refused(DZ_ESTATE, c.gqa_prefill_q4, 0, [1, 0], [0, 6], q, k, v, out)
    refused(DZ_EINVAL, c.gqa_prefill_q4, 0, [1, 1], [3, 3], q, k, v, out)
    refused(DZ_EINVAL, c.gqa_prefill_q4, 0, [1, 0], [7, -1], q, k, v, out)
    refused(DZ_EINVAL, c.gqa_prefill_q4, 0, [1], [0], q[:0], k[:0], v[:0], out[:0])
    refused(DZ_EINVAL, c.gqa_prefill_q4, 0, [2], [6], q, k, v, out)
    refused(DZ_EINVAL, c.gqa_prefill_q4, 0, [1], [5], q, k, v, out)              # 6 rows for 5 tokens
    refused(DZ_EINVAL, c.gqa_prefill_q4, 0, [1], [6], q, k.bfloat16(), v, out)
    refused(DZ_EINVAL, c.gqa_prefill_q4, 0, [1], [6], q, k, v, out, pos=torch.zeros(6, 3, device="cuda"))
    assert c.kv_len(0, 0) == 15 and c.kv_len(0, 1) == 0
    check(m, [1, 0], [1, 5])
    m.done()
