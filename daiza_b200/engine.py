"""Host-side mirror of Daiza's per-layer forward and cache interfaces.

Reference interfaces (guang384/Daiza, Daiza-engine/src):
  model/attention.rs:56-63   attention_forward_into(h, w, cfg, kv_cache, (cos, sin), ws)
  model/ssm.rs:425-431       ssm_forward_into(h, w, cfg, state, ws)
  cache/kv_cache.rs:16-130   KvCache {len, append, truncate, reset, from_raw}
  cache/ssm_state.rs:9-39    SsmState {state, conv_history, conv_head, reset}
  model/forward.rs:32-77     ModelState (owns one cache per layer)

The projections before and after the core are out of scope, so the forward
functions here take the projection outputs (q_gate/k/v, or qkv/alpha/beta/z)
and return the core's output (attn_out * sigmoid(gate), or the gated RMSNorm
y) -- exactly the tensors between the two Q1_0 GEMVs in the reference.

Device tensors are torch CUDA tensors (torch is used for device memory and
streams only); every computation runs in libdzattn.so.
"""
import ctypes as C
import os

import numpy as np

from . import _ffi
from ._ffi import check

HQ, HKV, GRP, HD, ROPE = 24, 4, 6, 256, 64
SSM_HK, SSM_HV, SSM_D, CONV_K = 16, 48, 128, 4
QKD, INNER = SSM_HK * SSM_D, SSM_HV * SSM_D
QKV_LEN = 2 * QKD + INNER
QG_ROW = 2 * HD


def _ptr(t):
    return C.c_void_p(t.data_ptr())


def _np_ptr(a):
    return a.ctypes.data_as(C.c_void_p)


def _stream(stream):
    import torch
    s = torch.cuda.current_stream() if stream is None else stream
    return C.c_void_p(s.cuda_stream)


def _tensor(name, t, dtype, numel, device=None):
    """Address of a contiguous CUDA tensor (on that device) that a 4-bit cache call takes; DZ_EINVAL otherwise."""
    if (t.get_device() == device or device is None and t.is_cuda) and t.dtype == dtype and t.is_contiguous() and \
            t.numel() == numel:
        return t.data_ptr()
    where = "CUDA" if device is None else f"cuda:{device}"
    raise _ffi.DzError(_ffi.DZ_EINVAL, f"{name} must be a contiguous {where} {dtype} tensor of {numel} values, got "
                                       f"{tuple(t.shape)} {t.dtype} on {t.device}, strides {t.stride()}")


_arrays = {}                                     # ctypes array types by (type, length)


def _ints(name, values, ctype, count=None):
    """ctypes array of whole numbers (a number, list or array); DZ_EINVAL if they do not fit or are not `count`.
    A list goes straight into the array: the numpy route costs as much as a small launch."""
    try:
        v = values if type(values) is list or type(values) is tuple else np.atleast_1d(values).tolist()
        n = len(v)
        if count is not None and n != count:
            raise ValueError(f"{count} numbers wanted, {n} given")
        top = 1 << 31 if ctype is C.c_int32 else 1 << 63
        if n and not (-top <= min(v) and max(v) < top):
            raise ValueError("out of range")
        array = _arrays.get((ctype, n))
        if array is None:
            array = _arrays[ctype, n] = ctype * n
        return array(*v)
    except (TypeError, ValueError) as e:
        raise _ffi.DzError(_ffi.DZ_EINVAL, f"{name}: {e}") from None


def _ids(seq_ids):
    return _ints("seq_ids", seq_ids, C.c_int32)


def _per_seq(name, values, ids):
    return _ints(name, values, C.c_int64, len(ids))


def _positions(pos, B):
    try:
        flat = [p for row in pos for p in row]
    except TypeError as e:
        raise _ffi.DzError(_ffi.DZ_EINVAL, f"pos is no [{B}][3]: {e}") from None
    return _ints("pos", flat, C.c_int32, 3 * B)


def _total(counts):
    """Sum of those of a ctypes array that are not negative (the call refuses the others)."""
    n = list(counts)
    return sum(n) if min(n, default=0) >= 0 else sum(c for c in n if c > 0)


def default_config(n_layers=64, full_attention_interval=4, kv_heads=None, v_heads=None, qtile_split=None):
    """Config::default (config.rs:47-74) with an optional head slice and
    GQA-prefill query-tile split (index, count)."""
    cfg = _ffi.dz_config()
    check(_ffi.lib().dz_config_default(C.byref(cfg)))
    cfg.n_layers = n_layers
    cfg.full_attention_interval = full_attention_interval
    if kv_heads is not None:
        cfg.kv_head_begin, cfg.kv_head_count = kv_heads[0], kv_heads[1] - kv_heads[0]
    if v_heads is not None:
        cfg.v_head_begin, cfg.v_head_count = v_heads[0], v_heads[1] - v_heads[0]
    if qtile_split is not None:
        cfg.qtile_split_index, cfg.qtile_split_count = qtile_split
    return cfg


class Context:
    """Owns the device caches of one GPU (ModelState, model/forward.rs:32-77)."""

    def __init__(self, device=0, config=None):
        self.lib = _ffi.lib()
        self.cfg = config if config is not None else default_config()
        h = C.c_void_p()
        st = self.lib.dz_ctx_create(int(device), C.byref(self.cfg), C.byref(h))
        if st != _ffi.DZ_OK:
            raise _ffi.DzError(st, f"dz_ctx_create(device={device}) failed")
        self.h = h
        self.device = device
        self.index = int(device)                     # what its tensors' get_device() gives
        self.kvc = self.cfg.kv_head_count
        self.vc = self.cfg.v_head_count
        self.nq = GRP * self.kvc

    def close(self):
        if self.h:
            self.lib.dz_ctx_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _chk(self, st):
        check(st, self.h)

    def is_attention(self, layer):
        return self.lib.dz_layer_is_attention(self.h, layer) == 1

    @property
    def last_launch_count(self):
        return self.lib.dz_last_launch_count(self.h)

    def device_error(self):
        code = C.c_int32(0)
        st = self.lib.dz_device_error(self.h, C.byref(code))
        return code.value if st in (_ffi.DZ_OK, _ffi.DZ_ETIMEOUT) else self._chk(st)

    # ---- parameters ------------------------------------------------------
    def set_attn_params(self, layer, q_norm, k_norm):
        q = np.ascontiguousarray(q_norm, np.float32)
        k = np.ascontiguousarray(k_norm, np.float32)
        self._chk(self.lib.dz_layer_set_attn_params(self.h, layer, _np_ptr(q), _np_ptr(k)))

    def set_ssm_params(self, layer, conv1d_t, ssm_a, dt_bias, ssm_norm):
        arrs = [np.ascontiguousarray(a, np.float32) for a in (conv1d_t, ssm_a, dt_bias, ssm_norm)]
        self._chk(self.lib.dz_layer_set_ssm_params(self.h, layer, *[_np_ptr(a) for a in arrs]))

    # ---- caches ----------------------------------------------------------
    def cache_create(self, max_len):
        ml = np.ascontiguousarray(np.atleast_1d(max_len), np.int64)
        self._chk(self.lib.dz_cache_create(self.h, len(ml), _np_ptr(ml)))
        self.n_seqs = len(ml)

    def kv_len(self, layer, seq):
        n = C.c_int64()
        self._chk(self.lib.dz_kv_len(self.h, layer, seq, C.byref(n)))
        return n.value

    def kv_lens(self, layer, seq_ids):
        """kv_len of several sequences, as a list."""
        ids = _ids(seq_ids)
        return list(self._lens(layer, ids))

    def _lens(self, layer, ids):
        out = _ints("lens", [0] * len(ids), C.c_int64)
        st = self.lib.dz_kv_lens(self.h, layer, len(ids), ids, out)
        if st != _ffi.DZ_OK:                     # the call takes a const context: it leaves no message there
            raise _ffi.DzError(st, f"no KV lengths of layer {layer}, seq_ids {list(ids)}")
        return out

    def kv_truncate(self, layer, seq, new_len):
        self._chk(self.lib.dz_kv_truncate(self.h, layer, seq, int(new_len)))

    def cache_reset(self, seq):
        self._chk(self.lib.dz_cache_reset(self.h, seq))

    # ---- Q1_0 projection GEMV ---------------------------------------------
    def q1_gemv(self, ws, x, ys, stream=None):
        """Q1_0Matrix::matvec_multi_into_slice for x [T][cols] (T <= 8) and up to
        8 Q1_0 matrices ws (uint8 device tensors [rows][cols/128*18]); writes
        ys[m] [T][rows]."""
        rows = np.array([w.shape[0] for w in ws], np.int32)
        cols = x.shape[-1]
        T = x.shape[0] if x.dim() == 2 else 1
        wp = (C.c_void_p * len(ws))(*[w.data_ptr() for w in ws])
        yp = (C.c_void_p * len(ys))(*[y.data_ptr() for y in ys])
        self._chk(self.lib.dz_q1_gemv(self.h, len(ws), C.cast(wp, C.c_void_p), _np_ptr(rows), cols, T, _ptr(x),
                                      C.cast(yp, C.c_void_p), _stream(stream)))

    def q1_gemv_add(self, ws, x, ys, stream=None):
        """matvec_add_into_slice: ys[m] += ws[m] x (same arguments as q1_gemv)."""
        rows = np.array([w.shape[0] for w in ws], np.int32)
        cols = x.shape[-1]
        T = x.shape[0] if x.dim() == 2 else 1
        wp = (C.c_void_p * len(ws))(*[w.data_ptr() for w in ws])
        yp = (C.c_void_p * len(ys))(*[y.data_ptr() for y in ys])
        self._chk(self.lib.dz_q1_gemv_add(self.h, len(ws), C.cast(wp, C.c_void_p), _np_ptr(rows), cols, T, _ptr(x),
                                          C.cast(yp, C.c_void_p), _stream(stream)))

    def rmsnorm_rows(self, x, w, out, stream=None):
        """math::rmsnorm_into per row of x [T][n] into out (the context's rms_eps)."""
        T, n = x.shape
        self._chk(self.lib.dz_rmsnorm_rows(self.h, T, n, _ptr(x), _ptr(w), _ptr(out), _stream(stream)))

    def block_mlp(self, h, post_norm_w, w_gate, w_up, w_down, stream=None):
        """block.rs:93-124 + mlp.rs:28-51 on h [T][hidden] in place."""
        T, hidden = h.shape
        d_ff = w_gate.shape[0]
        self._chk(self.lib.dz_block_mlp(self.h, T, hidden, d_ff, _ptr(h), _ptr(post_norm_w), _ptr(w_gate),
                                        _ptr(w_up), _ptr(w_down), _stream(stream)))

    # ---- DZSS session files ------------------------------------------------
    def session_save(self, seq, path, pos, history=(), think_enabled=False, system_prompt=None):
        """Session::save_to_disk (Daiza-runtime/src/session_persist.rs:76-140) for one sequence."""
        h = np.ascontiguousarray(np.asarray(history, np.uint32))
        sp = None if system_prompt is None else system_prompt.encode("utf-8")
        self._chk(self.lib.dz_session_save(self.h, int(seq), os.fspath(path).encode(), int(pos),
                                           _np_ptr(h) if h.size else None, int(h.size), int(bool(think_enabled)),
                                           sp))

    def session_load(self, seq, path, history_cap=1 << 20, prompt_cap=1 << 20):
        """Session::load_from_disk (session_persist.rs:186-290) into sequence seq;
        returns pos, history tokens, think flag and system prompt (or None)."""
        pos, n_hist, think, plen = C.c_int64(), C.c_int64(), C.c_int(), C.c_int64()
        hist = np.zeros(max(1, history_cap), np.uint32)
        buf = C.create_string_buffer(max(1, prompt_cap))
        self._chk(self.lib.dz_session_load(self.h, int(seq), os.fspath(path).encode(), C.byref(pos), _np_ptr(hist),
                                           int(history_cap), C.byref(n_hist), C.byref(think), buf, int(prompt_cap),
                                           C.byref(plen)))
        prompt = None if plen.value < 0 else buf.raw[:plen.value].decode("utf-8", "replace")
        return {"pos": pos.value, "history": hist[:n_hist.value].copy(), "think_enabled": bool(think.value),
                "system_prompt": prompt}

    # ---- sequence snapshots (speculative rollback) ------------------------
    def snapshot_reserve(self, n_slots):
        """Device memory for n_slots snapshots of one sequence's recurrent state."""
        self._chk(self.lib.dz_snapshot_reserve(self.h, int(n_slots)))

    def snapshot_save(self, seq, slot, stream=None):
        """DeltaNet states, conv rings and heads of every layer plus the KV lengths."""
        self._chk(self.lib.dz_snapshot_save(self.h, int(seq), int(slot), _stream(stream)))

    def snapshot_restore(self, seq, slot, stream=None):
        """Back to the saved state; KV lengths truncated to the saved ones."""
        self._chk(self.lib.dz_snapshot_restore(self.h, int(seq), int(slot), _stream(stream)))

    def kv_export(self, layer, seq):
        n = self.kv_len(layer, seq)
        k = np.zeros((n, self.kvc, HD), np.float32)
        v = np.zeros((n, self.kvc, HD), np.float32)
        self._chk(self.lib.dz_kv_export(self.h, layer, seq, _np_ptr(k), _np_ptr(v)))
        return k, v

    def kv_import(self, layer, seq, k_flat, v_flat):
        """k_flat, v_flat: [len][kvc][256] f32, numpy (host) or contiguous torch CUDA tensors."""
        if hasattr(k_flat, "data_ptr"):
            assert k_flat.is_contiguous() and v_flat.is_contiguous()
            self._chk(self.lib.dz_kv_import(self.h, layer, seq, _ptr(k_flat), _ptr(v_flat), k_flat.shape[0]))
            return
        k = np.ascontiguousarray(k_flat, np.float32)
        v = np.ascontiguousarray(v_flat, np.float32)
        self._chk(self.lib.dz_kv_import(self.h, layer, seq, _np_ptr(k), _np_ptr(v), k.shape[0]))

    def ssm_export(self, layer, seq):
        s = np.zeros((self.vc, SSM_D, SSM_D), np.float32)
        hst = np.zeros((CONV_K, QKV_LEN), np.float32)
        head = C.c_int32()
        self._chk(self.lib.dz_ssm_export(self.h, layer, seq, _np_ptr(s), _np_ptr(hst), C.byref(head)))
        return s, hst, head.value

    def ssm_import(self, layer, seq, state, conv_history, conv_head):
        if hasattr(state, "data_ptr"):
            self._chk(self.lib.dz_ssm_import(self.h, layer, seq, _ptr(state), _ptr(conv_history), int(conv_head)))
            return
        s = np.ascontiguousarray(state, np.float32)
        hst = np.ascontiguousarray(conv_history, np.float32)
        self._chk(self.lib.dz_ssm_import(self.h, layer, seq, _np_ptr(s), _np_ptr(hst), int(conv_head)))

    def kv_fill_pattern(self, layer, seq, length, byte_value=0x3C):
        """Synthetic KV rows (benchmarks): every byte of rows [0, length) = byte_value."""
        self._chk(self.lib.dz_kv_fill_pattern(self.h, layer, seq, int(length), int(byte_value)))

    def rope_table(self, pos0, n):
        out = np.zeros((n, 2 * ROPE), np.float32)
        self._chk(self.lib.dz_rope_table(self.h, int(pos0), int(n), _np_ptr(out)))
        return out

    def kv_cache(self, layer, seq):
        return KvCacheView(self, layer, seq)

    def ssm_state(self, layer, seq):
        return SsmStateView(self, layer, seq)

    # ---- compute (device tensors) ------------------------------------------
    def gqa_decode(self, layer, seq_ids, q_gate, k, v, out, stream=None, pos=None):
        """pos: RoPE positions of the new tokens (ModelState::pos); default = cache lengths."""
        ids = np.ascontiguousarray(np.atleast_1d(seq_ids), np.int32)
        if pos is None:
            self._chk(self.lib.dz_gqa_decode(self.h, layer, len(ids), _np_ptr(ids), _ptr(q_gate), _ptr(k), _ptr(v),
                                             _ptr(out), _stream(stream)))
            return
        ps = np.ascontiguousarray(np.atleast_1d(pos), np.int32)
        assert ps.shape == ids.shape
        self._chk(self.lib.dz_gqa_decode_at(self.h, layer, len(ids), _np_ptr(ids), _np_ptr(ps), _ptr(q_gate), _ptr(k),
                                            _ptr(v), _ptr(out), _stream(stream)))

    # ---- KV caches held in 4 bits -------------------------------------------
    def cache_create_q4(self, max_len, track=False):
        """cache_create with K and V held in 4 bits; track: accumulate attention weights."""
        ml = np.ascontiguousarray(np.atleast_1d(max_len), np.int64)
        self._chk(self.lib.dz_cache_create_q4(self.h, len(ml), _np_ptr(ml), int(bool(track))))
        self.n_seqs = len(ml)

    def set_rope_axes(self, sections=(11, 11, 10), interleaved=False):
        """Which of a token's (time, height, width) positions turns each of the 32 rotary pairs."""
        s = _ints("sections", sections, C.c_int32, 3)
        self._chk(self.lib.dz_set_rope_axes(self.h, s, int(bool(interleaved))))

    def _on(self, stream):
        """Handle of `stream`, or of the context's device's current one (straight, where this torch has the call for it:
        making a Stream object takes 1.3 us)."""
        if stream is not None:
            return stream.cuda_stream
        import torch
        raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        return raw(self.index) if raw else torch.cuda.current_stream(self.index).cuda_stream

    def qk_mrope(self, layer, pos, q_gate, k, q_out, k_out, stream=None):
        """QK-RMSNorm, rotation by pos [T][3] (int32) and q's 1/16; q_gate [T][6*kvc][512] and k [T][kvc][256] f32 or
        bf16, q_out [T][6*kvc][256] and k_out [T][kvc][256] of the same type."""
        import torch
        T = k.numel() // (self.kvc * HD)
        dt = torch.bfloat16 if k.dtype == torch.bfloat16 else torch.float32
        fn = self.lib.dz_qk_mrope_bf16 if dt == torch.bfloat16 else self.lib.dz_qk_mrope
        self._chk(fn(self.h, layer, T, _tensor("pos", pos, torch.int32, 3 * T, self.index),
                     _tensor("q_gate", q_gate, dt, T * self.nq * QG_ROW, self.index),
                     _tensor("k", k, dt, T * self.kvc * HD, self.index),
                     _tensor("q_out", q_out, dt, T * self.nq * HD, self.index),
                     _tensor("k_out", k_out, dt, T * self.kvc * HD, self.index), self._on(stream)))

    def gqa_decode_q4(self, layer, seq_ids, q_gate, k, v, out, stream=None, pos=None):
        """gqa_decode on 4-bit caches; pos: [B][3] rotary positions (host), default the cache lengths."""
        import torch
        ids, f = _ids(seq_ids), torch.float32
        B, p3 = len(ids), None
        if pos is not None:
            p3 = _positions(pos, B)
        self._chk(self.lib.dz_gqa_decode_q4(
            self.h, layer, B, ids, p3,
            _tensor("q_gate", q_gate, f, B * self.nq * QG_ROW, self.index),
            _tensor("k", k, f, B * self.kvc * HD, self.index), _tensor("v", v, f, B * self.kvc * HD, self.index),
            _tensor("out", out, f, B * self.nq * HD, self.index), self._on(stream)))

    def gqa_prefill_q4(self, layer, seq_ids, lens, q_gate, k, v, out, stream=None, pos=None):
        """lens[i] new tokens of each sequence, packed: q_gate [sum][6*kvc][512], k and v [sum][kvc][256], out
        [sum][6*kvc*256], all f32 or all bf16; pos: int32 CUDA tensor [sum][3], default the cache slots."""
        import torch
        ids = _ids(seq_ids)
        n = _per_seq("lens", lens, ids)
        T = _total(n)
        dt = torch.bfloat16 if k.dtype == torch.bfloat16 else torch.float32
        fn = self.lib.dz_gqa_prefill_q4_bf16 if dt == torch.bfloat16 else self.lib.dz_gqa_prefill_q4
        self._chk(fn(self.h, layer, len(ids), ids, n,
                     None if pos is None else _tensor("pos", pos, torch.int32, 3 * T, self.index),
                     _tensor("q_gate", q_gate, dt, T * self.nq * QG_ROW, self.index),
                     _tensor("k", k, dt, T * self.kvc * HD, self.index),
                     _tensor("v", v, dt, T * self.kvc * HD, self.index),
                     _tensor("out", out, dt, T * self.nq * HD, self.index), self._on(stream)))

    def kv_rows_q4(self, layer, seq_ids, first, count, k, v, stream=None):
        """Held rows [first, first + count) of each sequence as f32 [sum count][kvc][256]."""
        import torch
        ids = _ids(seq_ids)
        a, n = _per_seq("first", first, ids), _per_seq("count", count, ids)
        total = _total(n) * self.kvc * HD
        self._chk(self.lib.dz_kv_rows_q4(self.h, layer, len(ids), ids, a, n,
                                         _tensor("k", k, torch.float32, total, self.index),
                                         _tensor("v", v, torch.float32, total, self.index), self._on(stream)))

    def _weights_numel(self, layer, ids):
        return self.kvc * sum(self._lens(layer, ids))

    def kv_weights_q4(self, layer, seq_ids, out, stream=None):
        """Accumulated attention weights, sequence by sequence [kvc][length]."""
        import torch
        ids = _ids(seq_ids)
        self._chk(self.lib.dz_kv_weights_q4(
            self.h, layer, len(ids), ids,
            _tensor("out", out, torch.float32, self._weights_numel(layer, ids), self.index), self._on(stream)))

    def kv_set_weights_q4(self, layer, seq_ids, weights, stream=None):
        import torch
        ids = _ids(seq_ids)
        self._chk(self.lib.dz_kv_set_weights_q4(
            self.h, layer, len(ids), ids,
            _tensor("weights", weights, torch.float32, self._weights_numel(layer, ids), self.index), self._on(stream)))

    def kv_evict_q4(self, layer, seq_ids, keep, recent, kept=None, into=None, stream=None):
        """Keeps the last recent[b] and the heaviest other entries, keep[b] in all, per kv head; in place, or into the
        sequences `into`.  kept: int32 CUDA tensor, per sequence [kvc][min(keep, length)], their former rows."""
        import torch
        ids = _ids(seq_ids)
        k, r = _per_seq("keep", keep, ids), _per_seq("recent", recent, ids)
        to = None if into is None else _ints("into", into, C.c_int32, len(ids))
        out = None
        if kept is not None:
            n = sum(max(0, min(a, b)) for a, b in zip(k, self._lens(layer, ids)))
            out = _tensor("kept", kept, torch.int32, n * self.kvc, self.index)
        self._chk(self.lib.dz_kv_evict_q4(self.h, layer, len(ids), ids, to,
                                          k, r, out, self._on(stream)))

    def gdn_decode(self, layer, seq_ids, qkv, alpha, beta, z, y, stream=None):
        ids = np.ascontiguousarray(np.atleast_1d(seq_ids), np.int32)
        self._chk(self.lib.dz_gdn_decode(self.h, layer, len(ids), _np_ptr(ids), _ptr(qkv), _ptr(alpha), _ptr(beta),
                                         _ptr(z), _ptr(y), _stream(stream)))

    def gqa_prefill(self, layer, seq, q_gate, k, v, out, stream=None, start_pos=None):
        """start_pos: RoPE position of the first token (forward.rs:550-557); default = cache length."""
        import torch
        T = q_gate.shape[0]
        bf = q_gate.dtype == torch.bfloat16
        if start_pos is None:
            fn = self.lib.dz_gqa_prefill_bf16 if bf else self.lib.dz_gqa_prefill
            self._chk(fn(self.h, layer, seq, T, _ptr(q_gate), _ptr(k), _ptr(v), _ptr(out), _stream(stream)))
            return
        fn = self.lib.dz_gqa_prefill_bf16_at if bf else self.lib.dz_gqa_prefill_at
        self._chk(fn(self.h, layer, seq, int(start_pos), T, _ptr(q_gate), _ptr(k), _ptr(v), _ptr(out),
                     _stream(stream)))

    def gdn_prefill(self, layer, seq, qkv, alpha, beta, z, y, stream=None):
        T = qkv.shape[0]
        self._chk(self.lib.dz_gdn_prefill(self.h, layer, seq, T, _ptr(qkv), _ptr(alpha), _ptr(beta), _ptr(z),
                                          _ptr(y), _stream(stream)))

    # ---- compute (host arrays; end-to-end path) ----------------------------
    def gqa_decode_host(self, layer, seq_ids, q_gate, k, v, out=None, stream=None, sync=True):
        """sync=False: dz_gqa_decode_host_async -- the caller synchronises `stream`
        before reading `out` or reusing the inputs."""
        ids = np.ascontiguousarray(np.atleast_1d(seq_ids), np.int32)
        B = len(ids)
        if out is None:
            out = np.empty((B, self.nq * HD), np.float32)
        fn = self.lib.dz_gqa_decode_host if sync else self.lib.dz_gqa_decode_host_async
        self._chk(fn(self.h, layer, B, _np_ptr(ids), _np_ptr(q_gate), _np_ptr(k), _np_ptr(v), _np_ptr(out),
                     _stream(stream)))
        return out

    def gdn_decode_host(self, layer, seq_ids, qkv, alpha, beta, z, y=None, stream=None, sync=True):
        """sync=False: dz_gdn_decode_host_async (see gqa_decode_host)."""
        ids = np.ascontiguousarray(np.atleast_1d(seq_ids), np.int32)
        B = len(ids)
        if y is None:
            y = np.empty((B, self.vc * SSM_D), np.float32)
        fn = self.lib.dz_gdn_decode_host if sync else self.lib.dz_gdn_decode_host_async
        self._chk(fn(self.h, layer, B, _np_ptr(ids), _np_ptr(qkv), _np_ptr(alpha), _np_ptr(beta), _np_ptr(z),
                     _np_ptr(y), _stream(stream)))
        return y


class KvCacheView:
    """KvCache (cache/kv_cache.rs:16-130) of one (layer, sequence) in HBM."""

    def __init__(self, ctx, layer, seq):
        self.ctx, self.layer, self.seq = ctx, layer, seq

    @property
    def len(self):
        return self.ctx.kv_len(self.layer, self.seq)

    def truncate(self, new_len):
        self.ctx.kv_truncate(self.layer, self.seq, new_len)

    def to_raw(self):
        return self.ctx.kv_export(self.layer, self.seq)

    def load_raw(self, k_flat, v_flat):
        self.ctx.kv_import(self.layer, self.seq, k_flat, v_flat)


class SsmStateView:
    """SsmState (cache/ssm_state.rs:9-39) of one (layer, sequence) in HBM."""

    def __init__(self, ctx, layer, seq):
        self.ctx, self.layer, self.seq = ctx, layer, seq

    def export(self):
        return self.ctx.ssm_export(self.layer, self.seq)

    def load(self, state, conv_history, conv_head):
        self.ctx.ssm_import(self.layer, self.seq, state, conv_history, conv_head)


def attention_forward_into(ctx, layer, seq_ids, q_gate, k, v, out, stream=None):
    """Core of attention_forward_into (model/attention.rs:90-203) for a batch of sequences."""
    ctx.gqa_decode(layer, seq_ids, q_gate, k, v, out, stream)


def ssm_forward_into(ctx, layer, seq_ids, qkv, alpha, beta, z, y, stream=None):
    """Core of ssm_forward_into (model/ssm.rs:466-611) for a batch of sequences."""
    ctx.gdn_decode(layer, seq_ids, qkv, alpha, beta, z, y, stream)
