"""4-bit caches that are long for the kernels: runs of many tiles per warp in decode, running maxima that move at
several places, prompts behind long cached rows.  The restatement here is oracle/q4_ref.py's attention over the rows
that the cache holds (they are compared exactly elsewhere), in float64 on the GPU.

Tolerances as in test_gpu_q4.py and test_gpu_q4_prefill.py, with what a test adds to them beside it."""
import numpy as np
import pytest

from oracle import q4_ref as R
from tests.test_gpu_q4 import OUT_TOL, W_TOL, Model, dev
from tests.test_gpu_q4_prefill import MAX_TOL, NORM_TOL

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def held(m, seq):
    n = m.ctx.kv_len(0, seq)
    k, v = (torch.empty(n, m.kvc, 256, device="cuda") for _ in "kv")
    m.ctx.kv_rows_q4(0, [seq], [0], [n], k, v)
    return k.double(), v.double()


def attention(m, seq, q_gate, pos):
    """Output [T][heads][256] of the last T = len(pos) rows' tokens over the held rows, and the probabilities' sums
    [kv heads][length] over tokens and heads."""
    k, v = held(m, seq)
    n, T = len(k), len(pos)
    qg = torch.as_tensor(q_gate, device="cuda").double()
    q = torch.tensor(R.turn(qg[..., :256].cpu().numpy(), m.qn, pos, m.axis) / 16, device="cuda")
    later = torch.ones(T, n, dtype=torch.bool, device="cuda").triu(n - T + 1)
    out = torch.empty(T, m.nq, 256, device="cuda", dtype=torch.float64)
    w = torch.zeros(m.kvc, n, device="cuda", dtype=torch.float64)
    for i in range(m.nq):
        p = torch.softmax((q[:, i] @ k[:, i // 6].T).masked_fill(later, -np.inf), -1)
        out[:, i] = p @ v[:, i // 6]
        w[i // 6] += p.sum(0)
    return out * torch.sigmoid(qg[..., 256:]), w


def at(first, T):
    return np.repeat(np.arange(first, first + T)[:, None], 3, 1)


def stairs(n, width=128, steps=4, height=10.0):
    """Scores in log2 units that rise by `height` every `width` positions, `steps` levels, over and over."""
    return height * ((np.arange(n) // width) % steps)


def steep_keys(m, n, q, heads):
    """K rows [n][kvc][256] whose scores with the rotated query q [6 kvc][256] of the given heads are the stairs (each
    head's begin at another place), beside noise."""
    k = 0.3 * torch.randn(n, m.kvc, 256, device="cuda")
    for i in heads:
        a = np.roll(stairs(n), 37 * i) * np.log(2.0)
        k[:, i // 6] += torch.tensor(a, device="cuda", dtype=torch.float32)[:, None] * dev(q[i] / (q[i] @ q[i]))
    return k


@pytest.mark.parametrize("steep", [False, True])
@pytest.mark.parametrize("track", [False, True])
def test_decode_runs_of_many_tiles(track, steep):
    """Nine sequences of 13000-41000 positions: 50 to 60 tiles to a warp's run, its ring of three pairs refilled many
    times, runs that end in the middle of a row and go on in the next.  Steep: a running maximum outgrows what P holds
    every 128 positions, in some of the heads."""
    lens = [40961, 13007, 29999, 31, 35000, 20480, 16, 38111, 27003]
    m = Model([n + 2 for n in lens], kvc=4, seed=300, track=track)
    torch.manual_seed(300)
    qg, k, v = m.inputs(len(lens))
    for s, n in enumerate(lens):
        q = R.turn(qg[s:s + 1, :, :256], m.qn, at(n, 1))[0] / 16
        old = steep_keys(m, n, q, (0, 1, 7, 13, 23) if steep else ())
        m.ctx.kv_import(0, s, old, torch.randn(n, 4, 256, device="cuda"))
    for step in range(2):
        out = torch.empty(len(lens), m.nq * 256, device="cuda")
        before = m.weights(list(range(len(lens)))) if track else None
        m.ctx.gqa_decode_q4(0, list(range(len(lens))), dev(qg), dev(k), dev(v), out)
        after = m.weights(list(range(len(lens)))) if track else None
        for s, n in enumerate(lens):
            want, w = attention(m, s, qg[s:s + 1], at(n + step, 1))
            top = held(m, s)[1].abs().max()
            # steep scores reach 30 log2 units: f32 sums of 256 products of up to 21 in all, as the 16 of normalised rows
            err = (out[s].reshape(1, m.nq, 256).double() - want).abs().max()
            assert err <= (2.0 if steep else 1.0) * OUT_TOL * top, f"step {step} seq {s}: {err / top:.2e}"
            if track:
                new = after[s].astype(np.float64)
                new[:, :-1] -= before[s]
                w = w.cpu().numpy()
                # the sum so far is rounded by 2^-24 of itself
                slack = np.pad(2.0 ** -23 * before[s], ((0, 0), (0, 1)))
                assert np.all(np.abs(new - w) <= (2.0 if steep else 1.0) * W_TOL * np.maximum(w, w.mean()) + slack), f"seq {s}"
        qg = qg.copy()
        qg[..., 256:] = m.normal(len(lens), m.nq, 256)
    m.done()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_prompt_whose_maxima_move(dtype):
    """Scores rise by 10 log2 units every 128 keys for some heads and a third of the tokens: what has been summed up is
    scaled down at several key blocks, in some rows of a warp."""
    dt, T, base = getattr(torch, dtype), 200, 1500
    m = Model([base + T], kvc=2, seed=301)
    torch.manual_seed(301)
    qg, k, v = m.inputs(T)
    pos = np.zeros((T, 3), np.int64)                  # no rotation: tokens can share their queries
    common = m.normal(m.nq, 256)
    qg[::3, :, :256] = common
    qg, k, v = (dev(x, dt) for x in (qg, k, v))
    q = R.turn(qg[:1, :, :256].double().cpu().numpy(), m.qn, pos[:1])[0] / 16
    m.ctx.kv_import(0, 0, steep_keys(m, base, q, (0, 3, 8, 11)), torch.randn(base, 2, 256, device="cuda"))
    out = torch.empty(T, m.nq * 256, device="cuda", dtype=dt)
    m.ctx.gqa_prefill_q4(0, [0], [T], qg, k, v, out, pos=dev(pos, torch.int32))
    want, _ = attention(m, 0, qg, pos)
    got, top = out.double().reshape(want.shape), held(m, 0)[1].abs().max()
    step = 2.0 ** -8 if dtype == "bfloat16" else 0.0
    assert ((got - want).abs() <= MAX_TOL * top + step * want.abs()).all()
    # a score of 21 is the sum of 256 rounded products of one sign: its error 21 * 2^-12.3 / 16 = 2.6e-4 rms, as a normalised row's
    assert (got - want).norm() <= (1.5 * NORM_TOL + step / 3 ** 0.5) * want.norm()
    m.done()


@pytest.mark.parametrize("base,T,dtype", [(20000, 130, "float32"), (131000, 3, "float32"), (131000, 140, "bfloat16")])
def test_prompt_behind_long_cached_rows(base, T, dtype):
    """Values around 1, which add up in one direction: the matrix instruction truncates, up to 4 * 2^-23 of the sum at each
    of its additions of 16 keys; over a stretch of 8192 keys, along which the sum grows from 0, that is at most
    512 / 2 * 4 * 2^-23 = 1.2e-4 of it, whatever the length."""
    dt = getattr(torch, dtype)
    m = Model([base + T], kvc=1, seed=302)
    torch.manual_seed(302)
    m.ctx.kv_import(0, 0, torch.randn(base, 1, 256, device="cuda"), 1 + 0.1 * torch.randn(base, 1, 256, device="cuda"))
    qg, k, v = (dev(x, dt) for x in m.inputs(T))
    v = (1 + 0.1 * v.float()).to(dt)
    out = torch.empty(T, m.nq * 256, device="cuda", dtype=dt)
    m.ctx.gqa_prefill_q4(0, [0], [T], qg, k, v, out)
    want, _ = attention(m, 0, qg, at(base, T))
    got = out.double().reshape(want.shape)
    bias = (got / want - 1).mean().item()
    assert abs(bias) <= 1.2e-4, f"{bias:.2e}"
    step = 2.0 ** -8 / 3 ** 0.5 if dtype == "bfloat16" else 0.0
    top, err = held(m, 0)[1].abs().max(), (got - want).abs()
    assert (err <= MAX_TOL * top + (2.0 ** -8 * want.abs() if step else 0.0)).all(), err.max()
    assert err.norm() <= (NORM_TOL + step) * want.norm()
    m.done()


def test_prompt_behind_long_rows_of_very_low_scores():
    """All scores of a head far below 0 (log2 units -160 to -190), and rising from stretch to stretch in others."""
    base, T = 25000, 40
    m = Model([base + T], kvc=1, seed=304)
    torch.manual_seed(304)
    qg, k, v = m.inputs(T)
    pos = np.zeros((T, 3), np.int64)
    qg[:] = qg[:1]
    q = R.turn(qg[:1, :, :256], m.qn, pos[:1])[0] / 16
    u = q[0] / (q[0] @ q[0])
    old = dev(-120 * u).repeat(base, 1, 1) + 0.1 * torch.randn(base, 1, 256, device="cuda")
    w = q[3] - (q[3] @ q[0]) / (q[0] @ q[0]) * q[0]
    old += torch.arange(base, device="cuda")[:, None, None] / base * dev(40 * w / (w @ w))
    k[:] = 0
    m.kn[:] = 0                                       # the new keys' scores are 0: heads of low scores see them alone
    m.ctx.set_attn_params(0, m.qn, m.kn)
    m.ctx.kv_import(0, 0, old, torch.randn(base, 1, 256, device="cuda"))
    out = torch.empty(T, m.nq * 256, device="cuda")
    m.ctx.gqa_prefill_q4(0, [0], [T], dev(qg), dev(k), dev(v), out, pos=dev(pos, torch.int32))
    want, _ = attention(m, 0, qg, pos)
    got, top = out.double().reshape(want.shape), held(m, 0)[1].abs().max()
    # scores of up to 120: Q's rounding, 2^-12.3 / 16 of their size for keys along the query, 1.4e-3, 4 sigma in a probability
    assert (got - want).abs().max() <= (MAX_TOL + 4 * 120 * 2.0 ** -12.3 / 16) * top
    m.done()


def test_prompt_long_tail_behind_one_heavy_key():
    """One key 25 to 26 log2 units above 200000 others, whose weights together are about 0.4 %."""
    base, T = 200000, 2
    m = Model([base + T], kvc=1, seed=303)
    qg, k, v = m.inputs(T)
    pos = np.zeros((T, 3), np.int64)
    qg[:] = qg[:1, :1]
    q = R.turn(qg[:1, :1, :256], m.qn, pos[:1])[0, 0] / 16
    old = torch.zeros(base, 1, 256, device="cuda")
    heavy = R.hold(25.5 * np.log(2.0) * q / (q @ q))
    assert 25.1 < heavy @ q / np.log(2.0) < 25.9
    old[0, 0] = dev(heavy)
    values = torch.ones(base, 1, 256, device="cuda")
    values[0] = 0
    m.ctx.kv_import(0, 0, old, values)
    out = torch.empty(T, m.nq * 256, device="cuda")
    m.ctx.gqa_prefill_q4(0, [0], [T], dev(qg), dev(k), dev(v), out, pos=dev(pos, torch.int32))
    want, _ = attention(m, 0, qg, pos)
    got = out.double().reshape(want.shape)
    # P of the tail is 2^-18.5 or so, with f16's steps of 2^-24 there: within 2 %
    assert ((got - want).abs() <= 0.02 * want.abs() + 1e-5).all(), ((got - want).abs() / want.abs()).max()
    m.done()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_long_and_short_prompts_packed_split_and_replayed(dtype):
    """A prompt behind 9001 rows among short ones: in one call, as two contexts that share the query tiles, and in a graph
    that is replayed."""
    import daiza_b200 as dz
    dt, bases, lens = getattr(torch, dtype), [0, 9001, 300], [140, 300, 5]
    caps = [a + b for a, b in zip(bases, lens)]
    m = Model(caps, kvc=1, seed=305, track=True)
    torch.manual_seed(305)
    old = [torch.randn(2, n, 1, 256, device="cuda") for n in bases]
    qg, k, v = (dev(x, dt) for x in m.inputs(sum(lens)))

    def load(ctx):
        for s, n in enumerate(bases):
            ctx.kv_import(0, s, old[s][0], old[s][1])

    def run(ctx, out):
        ctx.gqa_prefill_q4(0, [0, 1, 2], lens, qg, k, v, out)

    load(m.ctx)
    whole = torch.empty(sum(lens), m.nq * 256, device="cuda", dtype=dt)
    run(m.ctx, whole)
    a, step = 0, 2.0 ** -8 if dtype == "bfloat16" else 0.0
    for s, n in enumerate(lens):
        want, _ = attention(m, s, qg[a:a + n], at(bases[s], n))
        got = whole[a:a + n].double().reshape(want.shape)
        assert ((got - want).abs() <= MAX_TOL * held(m, s)[1].abs().max() + step * want.abs()).all(), s
        assert (got - want).norm() <= (NORM_TOL + step / 3 ** 0.5) * want.norm(), s
        a += n
    halves = torch.full_like(whole, -7.0)
    for i in range(2):
        c = dz.Context(0, dz.default_config(n_layers=1, full_attention_interval=1, kv_heads=(0, 1), qtile_split=(i, 2)))
        c.set_attn_params(0, m.qn, m.kn)
        c.cache_create_q4(caps)
        load(c)
        run(c, halves)
        torch.cuda.synchronize()
        c.close()
    assert torch.equal(halves, whole)
    for s, n in enumerate(bases):
        m.ctx.kv_truncate(0, s, n)
    again = torch.empty_like(whole)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(m.ctx, again)
    for _ in range(2):
        again.fill_(-7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(again, whole)
    m.done()
