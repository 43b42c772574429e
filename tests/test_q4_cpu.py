"""4-bit KV cache, what needs no GPU: properties of the row format (oracle/q4_ref.py) and
refusals that come before any device work."""
import ctypes as C

import numpy as np
import pytest

from oracle import q4_ref as R


def rows(seed, n=64, spread=3.0):
    r = np.random.default_rng(seed)
    return r.standard_normal((n, 256)) * np.exp(spread * r.standard_normal((n, 1)))


def test_held_values_are_f16_with_few_bits():
    """code * scale is exact in f16, and 72 * scale (the unpacking's constant) is one too."""
    _, s = R.codes(np.concatenate([rows(1), rows(2) * 1e4, rows(3) * 1e-6]))
    held = R.hold(rows(1))
    assert np.array_equal(held, held.astype(np.float16).astype(np.float64))
    for k in (1, 7, 72):
        assert np.array_equal(k * s, (k * s).astype(np.float16).astype(np.float64))
    assert np.all((s.astype(np.float16).view(np.uint16) & 127) == 0)     # 8 bits hold it


def test_error_is_half_a_step_and_holding_again_changes_nothing():
    x = rows(4, spread=1.0)                          # nothing near the largest held value
    c, s = R.codes(x)
    held = R.hold(x)
    normal = np.repeat(s, 32, -1) >= 2.0 ** -14
    assert np.all((np.abs(x - held) <= np.repeat(s, 32, -1) / 2)[normal])
    assert np.abs(c).max() == 7
    for v in (held, R.hold(1e-6 * x), R.hold(1e5 * x)):
        assert np.array_equal(R.hold(v), v)


def test_ties_zeros_and_what_is_not_finite():
    x = np.zeros((3, 256))
    x[0, :4] = [7.0, 0.5, 1.5, -2.5]                 # scale 1: ties go to the even code
    x[1, :3] = [np.nan, np.inf, -np.inf]
    x[2, 0] = 2.0 ** -30                             # below half the smallest scale
    assert R.hold(x)[0, :4].tolist() == [7.0, 0.0, 2.0, -2.0]
    assert R.hold(x)[1, :3].tolist() == [0.0, 7 * 896.0, -7 * 896.0]
    assert not R.hold(x)[2].any()


def test_axes_of_the_rotary_pairs():
    assert np.bincount(R.axes()).tolist() == [11, 11, 10]
    assert np.bincount(R.axes(interleaved=True)).tolist() == [11, 11, 10]
    assert R.axes(interleaved=True)[:6].tolist() == [0, 1, 2, 0, 1, 2]
    assert R.axes((16, 8, 8), True)[24:].tolist() == [0, 0, 0, 0, 0, 0, 0, 0]


def test_prompt_is_its_tokens_one_by_one():
    r = np.random.default_rng(5)
    qg, k, v = r.standard_normal((5, 6, 512)), r.standard_normal((5, 1, 256)), r.standard_normal((5, 1, 256))
    qn, kn = 1 + 0.1 * r.standard_normal((2, 256))
    whole, steps = R.Cache(1), R.Cache(1)
    a = whole.extend(qg, k, v, qn, kn)
    b = np.concatenate([steps.extend(qg[t:t + 1], k[t:t + 1], v[t:t + 1], qn, kn) for t in range(5)])
    assert np.array_equal(a, b) and np.array_equal(whole.w, steps.w)
    assert np.allclose(whole.w.sum(), 5 * 6)


def test_eviction_keeps_the_recent_and_the_heaviest():
    c = R.Cache(1, np.ones((6, 1, 256)), np.ones((6, 1, 256)))
    c.w = np.array([[0.5, 0.0, 0.5, 2.0, 0.5, 0.0]])
    assert c.evict(4, 1).tolist() == [[0, 2, 3, 5]]          # of three equal weights the first two
    assert c.w.tolist() == [[0.5, 0.5, 2.0, 0.0]]
    assert c.evict(9, 1).tolist() == [[0, 1, 2, 3]]


def test_null_contexts_are_refused():
    from daiza_b200 import _ffi
    lib, none = _ffi.lib(), None
    sections = (C.c_int32 * 3)(11, 11, 10)
    one = (C.c_int64 * 1)(4)
    ids = (C.c_int32 * 1)(0)
    assert lib.dz_cache_create_q4(none, 1, one, 0) == _ffi.DZ_EINVAL
    assert lib.dz_set_rope_axes(none, sections, 0) == _ffi.DZ_EINVAL
    assert lib.dz_qk_mrope(none, 0, 1, none, none, none, none, none, none) == _ffi.DZ_EINVAL
    assert lib.dz_qk_mrope_bf16(none, 0, 1, none, none, none, none, none, none) == _ffi.DZ_EINVAL
    assert lib.dz_gqa_decode_q4(none, 0, 1, ids, none, none, none, none, none, none) == _ffi.DZ_EINVAL
    assert lib.dz_gqa_prefill_q4(none, 0, 1, ids, one, none, none, none, none, none, none) == _ffi.DZ_EINVAL
    assert lib.dz_gqa_prefill_q4_bf16(none, 0, 1, ids, one, none, none, none, none, none, none) == _ffi.DZ_EINVAL
    assert lib.dz_kv_lens(none, 0, 1, ids, one) == _ffi.DZ_EINVAL
    assert lib.dz_kv_rows_q4(none, 0, 1, ids, one, one, none, none, none) == _ffi.DZ_EINVAL
    assert lib.dz_kv_evict_q4(none, 0, 1, ids, none, one, one, none, none) == _ffi.DZ_EINVAL
    assert lib.dz_kv_weights_q4(none, 0, 1, ids, none, none) == _ffi.DZ_EINVAL
    assert lib.dz_kv_set_weights_q4(none, 0, 1, ids, none, none) == _ffi.DZ_EINVAL


def test_host_tensors_wrong_types_and_sizes_are_refused():
    torch = pytest.importorskip("torch")
    from daiza_b200 import engine
    from daiza_b200._ffi import DZ_EINVAL, DzError
    for bad in (torch.zeros(4), torch.zeros(4, dtype=torch.bfloat16)):
        with pytest.raises(DzError) as e:
            engine._tensor("x", bad, torch.float32, 4)
        assert e.value.status == DZ_EINVAL
    for name, bad in (("too many", [1, 2]), ("not whole", [1.5]), ("too large", [1 << 63]), ("no number", ["a"])):
        with pytest.raises(DzError) as e:
            engine._per_seq(name, bad, engine._ids([0]))
        assert e.value.status == DZ_EINVAL
    with pytest.raises(DzError):
        engine._ids([1 << 31])
    assert list(engine._ids(np.array([3, 1]))) == [3, 1] and list(engine._ids(2)) == [2]
    assert list(engine._per_seq("count", (4, 5), engine._ids([0, 1]))) == [4, 5]


class OnGpu:
    """What the checks ask of a tensor, for one that lies on another GPU."""
    is_cuda, shape = True, (256,)

    def __init__(self, torch, index):
        self.dtype, self.index, self.device = torch.float32, index, f"cuda:{index}"

    def get_device(self):
        return self.index

    def is_contiguous(self):
        return True

    def numel(self):
        return 256

    def stride(self):
        return (1,)

    def data_ptr(self):
        return 4096


def test_tensors_of_another_gpu_are_refused():
    torch = pytest.importorskip("torch")
    from daiza_b200 import engine
    from daiza_b200._ffi import DZ_EINVAL, DzError
    here, there = OnGpu(torch, 0), OnGpu(torch, 1)
    assert engine._tensor("x", here, torch.float32, 256, 0) == 4096

    class Lib:
        called = 0

        def dz_kv_rows_q4(self, *a):
            self.called += 1
            return 0

    ctx = engine.Context.__new__(engine.Context)     # a context of cuda:0, as far as its checks go
    ctx.index, ctx.h, ctx.kvc, ctx.lib, ctx._on = 0, None, 1, Lib(), lambda stream: None
    ctx.kv_rows_q4(0, [0], [0], [1], here, here)
    for pair in ((here, there), (there, here)):
        with pytest.raises(DzError) as e:
            ctx.kv_rows_q4(0, [0], [0], [1], *pair)
        assert e.value.status == DZ_EINVAL and "cuda:0" in str(e.value)
    assert ctx.lib.called == 1


def test_what_is_no_list_of_numbers_is_refused():
    pytest.importorskip("torch")
    from daiza_b200 import engine
    from daiza_b200._ffi import DZ_EINVAL, DzError

    class OnAGpu:                                    # what numpy does with a CUDA tensor
        def __array__(self, *a, **kw):
            raise TypeError("cannot convert a CUDA tensor to numpy")

    for call in (lambda: engine._ids(OnAGpu()), lambda: engine._positions([1, 2, 3], 1),
                 lambda: engine._positions(7, 1), lambda: engine._positions([[1, 2], [3, 4]], 1),
                 lambda: engine._positions([[1, 2, 1 << 31]], 1)):
        with pytest.raises(DzError) as e:
            call()
        assert e.value.status == DZ_EINVAL
    assert list(engine._positions(np.array([[1, 2, 3]], np.int32), 1)) == [1, 2, 3]


def test_refused_lengths_say_what_was_asked_for():
    """dz_kv_lens has no place for a message, and the last one of the context is of another call."""
    pytest.importorskip("torch")
    from daiza_b200 import _ffi, engine
    ctx = engine.Context.__new__(engine.Context)
    ctx.lib, ctx.h = _ffi.lib(), None
    with pytest.raises(_ffi.DzError) as e:
        ctx.kv_lens(5, [7, 9])
    assert e.value.status == _ffi.DZ_EINVAL and "layer 5" in str(e.value) and "[7, 9]" in str(e.value)


def test_current_stream_without_torchs_private_call(monkeypatch):
    torch = pytest.importorskip("torch")
    from daiza_b200 import engine
    ctx = engine.Context.__new__(engine.Context)
    ctx.index, ctx.h = 3, None
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: 100 + device, raising=False)
    assert ctx._on(None) == 103
    monkeypatch.delattr(torch._C, "_cuda_getCurrentRawStream")

    class Stream:
        def __init__(self, device):
            self.cuda_stream = 200 + device

    monkeypatch.setattr(torch.cuda, "current_stream", Stream)
    assert ctx._on(None) == 203 and ctx._on(Stream(7)) == 207
