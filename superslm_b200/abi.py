"""ctypes binding of the `sslm_*` C ABI.

The same binding drives two libraries that export identical verbs:

* ``libsslm_b200.so`` -- this package's CUDA implementation (the product), and
* the reference's own CPU library (test infrastructure, loaded only by tests and
  by the CPU-baseline leg of the benchmark).

Verb names, argument order and status ordinals are the reference's
(include/superslm/sslm_abi.h:96-163, sslm_abi_functions.inc,
sslm_abi_functions_g5_comparable.inc). The higher-level `Engine` / `Sequence`
helpers below mirror how the reference's own ABI callers drive it
(tools/t2147_chunk_batched_pins.cpp:133-154): map, pool, workspace, sequence,
chunked prefill, per-call decode.
"""
from __future__ import annotations

import ctypes as C
import os
import struct

import numpy as np

SSLM_OK = 0
STATUS_NAMES = [
    "SSLM_OK", "SSLM_INVALID_ARGUMENT", "SSLM_BUFFER_TOO_SMALL", "SSLM_MISALIGNED_BUFFER",
    "SSLM_ARTIFACT_REJECTED", "SSLM_ADAPTER_MODEL_MISMATCH", "SSLM_RESTORE_MODEL_MISMATCH",
    "SSLM_RESTORE_KV_MISMATCH", "SSLM_MODEL_HAS_LIVE_SEQUENCES", "SSLM_POOL_HAS_LIVE_HANDLES",
    "SSLM_ADAPTER_HAS_LIVE_SEQUENCES", "SSLM_ADAPTER_SWAP_MIDTOKEN_REJECTED",
    "SSLM_SEQ_RESET_MIDTOKEN_REJECTED", "SSLM_PREFIX_FROZEN_REJECTED", "SSLM_KV_POOL_EXHAUSTED",
    "SSLM_TOKEN_ID_OUT_OF_RANGE", "SSLM_CONTEXT_CAP_EXCEEDED", "SSLM_TOKEN_ID_UNMAPPED",
    "SSLM_SCHEMA_NOT_FOUND", "SSLM_SCHEMA_BIND_REJECTED", "SSLM_SCHEMA_SPAN_UNBOUND",
    "SSLM_PREFIX_SCHEMA_MISMATCH", "SSLM_RESTORE_SCHEMA_MISMATCH", "SSLM_SCHEMA_SPAN_UNREACHABLE",
    "SSLM_SCHEMA_UNSATISFIABLE", "SSLM_ALLOCATION_FAILED", "SSLM_NUMERIC_STEP_REFUSED",
]
ST = {n: i for i, n in enumerate(STATUS_NAMES)}


class SslmConfig(C.Structure):
    _fields_ = [("max_batch", C.c_int32), ("max_chunk_budget", C.c_int32),
                ("max_layer_budget", C.c_int32), ("reserved", C.c_uint32)]


class SslmDecodeParams(C.Structure):
    _fields_ = [("layer_budget", C.c_int32), ("struct_size", C.c_uint32), ("mode", C.c_int32),
                ("alpha_q15", C.c_int32), ("anti_lm_max_order", C.c_int32), ("top_k", C.c_int32),
                ("q_ln2", C.c_int64), ("q_b", C.c_int64), ("q_c", C.c_int64)]


class SslmControls(C.Structure):
    _fields_ = [("struct_size", C.c_uint32), ("repetition", C.c_int32), ("presence", C.c_int32), ("frequency", C.c_int32),
                ("count_given", C.c_int32), ("n_bias", C.c_int32), ("bias_tokens", C.POINTER(C.c_int32)), ("bias_values", C.POINTER(C.c_int32))]


_H = C.c_void_p  # opaque handle


def _aligned_buffer(nbytes: int, align: int = 64):
    raw = (C.c_uint8 * (nbytes + align))()
    addr = C.addressof(raw)
    off = (-addr) % align
    return raw, C.c_void_p(addr + off)


class SslmLib:
    """One loaded library exporting the sslm_* verbs."""

    VERBS = {
        "sslm_model_map": (C.c_int, [C.c_void_p, C.c_size_t, C.POINTER(_H)]),
        "sslm_model_unmap": (C.c_int, [_H]),
        "sslm_kv_block_size": (C.c_size_t, [_H]),
        "sslm_kv_pool_overhead_size": (C.c_size_t, [_H, C.c_uint32]),
        "sslm_kv_pool_create": (C.c_int, [_H, C.c_void_p, C.c_size_t, C.c_uint32, C.POINTER(_H)]),
        "sslm_kv_pool_destroy": (C.c_int, [_H]),
        "sslm_workspace_size": (C.c_size_t, [_H, C.POINTER(SslmConfig)]),
        "sslm_workspace_create": (C.c_int, [_H, C.POINTER(SslmConfig), C.c_void_p, C.c_size_t, C.POINTER(_H)]),
        "sslm_workspace_destroy": (C.c_int, [_H]),
        "sslm_seq_create": (C.c_int, [_H, C.POINTER(_H), C.POINTER(_H)]),
        "sslm_seq_release": (C.c_int, [_H]),
        "sslm_prefill": (C.c_int, [_H, _H, C.POINTER(C.c_int32), C.c_int32, C.c_int32, C.c_int, _H,
                                   C.POINTER(C.c_int32)]),
        "sslm_decode_step": (C.c_int, [_H, C.POINTER(_H), C.c_int32, C.POINTER(SslmDecodeParams), _H,
                                       C.POINTER(C.c_int32)]),
        "sslm_adapter_map": (C.c_int, [C.c_void_p, C.c_size_t, _H, C.POINTER(_H)]),
        "sslm_adapter_release": (C.c_int, [_H]),
        "sslm_adapter_residency": (C.c_size_t, [_H]),
        "sslm_seq_set_adapter": (C.c_int, [_H, _H]),
        "sslm_seq_save": (C.c_int, [_H, C.c_void_p, C.POINTER(C.c_size_t)]),
        "sslm_seq_restore": (C.c_int, [_H, C.POINTER(_H), C.c_void_p, C.c_size_t, C.POINTER(_H)]),
        "sslm_seq_reset": (C.c_int, [_H]),
        "sslm_prefix_begin": (C.c_int, [_H, C.POINTER(_H), C.POINTER(_H)]),
        "sslm_prefix_prefill": (C.c_int, [_H, _H, C.POINTER(C.c_int32), C.c_int32, C.c_int32, C.c_int, _H,
                                          C.POINTER(C.c_int32)]),
        "sslm_prefix_freeze": (C.c_int, [_H]),
        "sslm_prefix_release": (C.c_int, [_H]),
        "sslm_seq_adopt_prefix": (C.c_int, [_H, _H]),
        "sslm_schema_lookup": (C.c_int, [_H, C.c_char_p, C.POINTER(_H)]),
        "sslm_schema_count": (C.c_size_t, [_H]),
        "sslm_schema_name": (C.c_int, [_H, C.c_int32, C.c_char_p, C.POINTER(C.c_size_t)]),
        "sslm_seq_set_schema": (C.c_int, [_H, _H]),
        "sslm_prefix_set_schema": (C.c_int, [_H, _H]),
    }

    def __init__(self, path: str):
        if not os.path.exists(path):
            raise FileNotFoundError(path)
        self.path = path
        self.dll = C.CDLL(path, mode=os.RTLD_LOCAL | os.RTLD_NOW)
        for name, (res, args) in self.VERBS.items():
            fn = getattr(self.dll, name)
            fn.restype = res
            fn.argtypes = args
            setattr(self, name, fn)


class SslmError(RuntimeError):
    def __init__(self, verb, status):
        self.status = status
        nm = STATUS_NAMES[status] if 0 <= status < len(STATUS_NAMES) else str(status)
        super().__init__("%s -> %s" % (verb, nm))


def _chk(verb, st):
    if st != SSLM_OK:
        raise SslmError(verb, st)


class DecodeBatch:
    """See Engine.batch."""

    def __init__(self, eng: "Engine", seqs, layer_budget: int):
        self.eng = eng
        self.n = len(seqs)
        self.arr = (_H * self.n)(*[s.handle for s in seqs])
        self.params = SslmDecodeParams(layer_budget=layer_budget)
        self.out = (C.c_int32 * self.n)()
        self.tokens = np.ctypeslib.as_array(self.out)
        self._call = eng.lib.sslm_decode_step
        self._params_ref = C.byref(self.params)

    def step(self) -> int:
        return self._call(self.eng.model, self.arr, self.n, self._params_ref, self.eng.ws, self.out)


class Engine:
    """model + kv pool + workspace over one library."""

    def __init__(self, lib: SslmLib, artifact: bytes, blocks: int = 1, max_batch: int = 1,
                 max_chunk: int = 64):
        self.lib = lib
        self._art = np.frombuffer(artifact, dtype=np.uint8)
        self.model = _H()
        _chk("sslm_model_map", lib.sslm_model_map(self._art.ctypes.data, self._art.size, C.byref(self.model)))
        self.block_size = lib.sslm_kv_block_size(self.model)
        need = self.block_size * blocks + lib.sslm_kv_pool_overhead_size(self.model, blocks)
        self._pool_raw, pool_ptr = _aligned_buffer(need)
        self.pool = _H()
        _chk("sslm_kv_pool_create",
             lib.sslm_kv_pool_create(self.model, pool_ptr, need, blocks, C.byref(self.pool)))
        layers = struct.unpack_from("<I", artifact, _config_offset(artifact) + 12)[0]
        self.num_layers = layers
        self.cfg = SslmConfig(max_batch, max_chunk, layers, 0)
        wsz = lib.sslm_workspace_size(self.model, C.byref(self.cfg))
        self._ws_raw, ws_ptr = _aligned_buffer(wsz)
        self.ws = _H()
        _chk("sslm_workspace_create",
             lib.sslm_workspace_create(self.model, C.byref(self.cfg), ws_ptr, wsz, C.byref(self.ws)))
        self.adapters = []
        self.seqs = []

    def new_seq(self) -> "Sequence":
        s = Sequence(self)
        self.seqs.append(s)
        return s

    def map_adapter(self, artifact: bytes):
        a = np.frombuffer(artifact, dtype=np.uint8)
        h = _H()
        _chk("sslm_adapter_map", self.lib.sslm_adapter_map(a.ctypes.data, a.size, self.model, C.byref(h)))
        self.adapters.append((h, a))
        return h

    def decode_step(self, seqs, layer_budget: int):
        """One sslm_decode_step over a batch; returns (status, tokens)."""
        n = len(seqs)
        arr = (_H * n)(*[s.handle for s in seqs])
        params = SslmDecodeParams(layer_budget=layer_budget)
        out = (C.c_int32 * n)()
        st = self.lib.sslm_decode_step(self.model, arr, n, C.byref(params), self.ws, out)
        return st, list(out)

    def batch(self, seqs, layer_budget: int):
        """A fixed batch prepared once, the way a C caller holds its handle array: step() is then
        just the sslm_decode_step call, and `tokens` is a numpy view of the output buffer."""
        return DecodeBatch(self, seqs, layer_budget)

    def close(self):
        for s in list(self.seqs):
            s.release()
        for h, _ in self.adapters:
            self.lib.sslm_adapter_release(h)
        self.adapters = []
        if self.ws:
            self.lib.sslm_workspace_destroy(self.ws)
            self.ws = None
        if self.pool:
            self.lib.sslm_kv_pool_destroy(self.pool)
            self.pool = None
        if self.model:
            self.lib.sslm_model_unmap(self.model)
            self.model = None


def _config_offset(artifact: bytes) -> int:
    nsec = struct.unpack_from("<I", artifact, 12)[0]
    for i in range(nsec):
        stype, _dt, off = struct.unpack_from("<IIQ", artifact, 64 + 40 * i)
        if stype == 0:
            return off
    raise ValueError("no Config section")


class Sequence:
    def __init__(self, eng: Engine):
        self.eng = eng
        self.handle = _H()
        _chk("sslm_seq_create", eng.lib.sslm_seq_create(eng.model, C.byref(eng.pool), C.byref(self.handle)))

    def prefill(self, tokens, chunk_budget: int) -> int:
        """Feed all tokens in calls of at most chunk_budget; returns tokens consumed."""
        toks = np.ascontiguousarray(tokens, dtype=np.int32)
        done = 0
        while done < toks.size:
            consumed = C.c_int32(0)
            ptr = toks[done:].ctypes.data_as(C.POINTER(C.c_int32))
            st = self.eng.lib.sslm_prefill(self.eng.model, self.handle, ptr, toks.size - done,
                                           chunk_budget, 0, self.eng.ws, C.byref(consumed))
            done += consumed.value
            _chk("sslm_prefill", st)
            if consumed.value == 0:
                break
        return done

    def decode(self, n_tokens: int, layer_budget: int):
        """Greedy decode n_tokens tokens, calling sslm_decode_step until each lands."""
        out = []
        while len(out) < n_tokens:
            st, toks = self.eng.decode_step([self], layer_budget)
            _chk("sslm_decode_step", st)
            if toks[0] >= 0:
                out.append(toks[0])
        return out

    def set_adapter(self, adapter_handle):
        _chk("sslm_seq_set_adapter", self.eng.lib.sslm_seq_set_adapter(self.handle, adapter_handle))

    def set_controls(self, repetition=32768, presence=0, frequency=0, count_given=False, biases=()):
        """sslm_b200_seq_set_controls: penalties for repeated tokens (repetition in Q15, the others in logit units) and biases, pairs of
        (token, value); repetition=None takes them away."""
        fn = self.eng.lib.dll.sslm_b200_seq_set_controls
        fn.restype, fn.argtypes = C.c_int, [_H, C.c_void_p]
        if repetition is None:
            _chk("sslm_b200_seq_set_controls", fn(self.handle, None))
            return
        biases = list(biases)
        tokens, values = ((C.c_int32 * len(biases))(*[b[i] for b in biases]) for i in range(2))
        c = SslmControls(C.sizeof(SslmControls), repetition, presence, frequency, int(count_given), len(biases),
                         C.cast(tokens, C.POINTER(C.c_int32)), C.cast(values, C.POINTER(C.c_int32)))
        _chk("sslm_b200_seq_set_controls", fn(self.handle, C.addressof(c)))

    def save(self) -> bytes:
        n = C.c_size_t(0)
        self.eng.lib.sslm_seq_save(self.handle, None, C.byref(n))
        buf = (C.c_uint8 * n.value)()
        _chk("sslm_seq_save", self.eng.lib.sslm_seq_save(self.handle, buf, C.byref(n)))
        return bytes(buf[:n.value])

    def reset(self):
        _chk("sslm_seq_reset", self.eng.lib.sslm_seq_reset(self.handle))

    @classmethod
    def restore(cls, eng: "Engine", blob: bytes) -> "Sequence":
        """A new sequence of `eng` from a save blob (either library's)."""
        s = cls.__new__(cls)
        s.eng = eng
        s.handle = _H()
        raw = np.frombuffer(blob, dtype=np.uint8)
        _chk("sslm_seq_restore", eng.lib.sslm_seq_restore(eng.model, C.byref(eng.pool), raw.ctypes.data, raw.size,
                                                          C.byref(s.handle)))
        eng.seqs.append(s)
        return s

    def release(self):
        if self.handle:
            self.eng.lib.sslm_seq_release(self.handle)
            self.handle = None
            if self in self.eng.seqs:
                self.eng.seqs.remove(self)


# ---- operators on tensors in GPU memory (sslm_b200_*_resident). A call is prepared once from the tensors of a
# program (anything with torch's data_ptr / shape / stride / dtype / device) and then run as often as their contents
# change, like a batch of Engine.batch. It holds the tensors, copies none of them and keeps no result.
class PrefixAttentionArgs(C.Structure):
    _fields_ = [("struct_size", C.c_uint32), ("rows", C.c_int32), ("groups", C.c_int32), ("heads", C.c_int32), ("kv_heads", C.c_int32),
                ("head_dim", C.c_int32), ("max_prefix", C.c_int32), ("max_suffix", C.c_int32), ("q", C.c_void_p), ("q_stride", C.c_int64),
                ("consts", C.c_void_p), ("kv", C.c_void_p), ("num_pages", C.c_int64), ("group_start", C.c_void_p), ("prefix_len", C.c_void_p),
                ("prefix_pages", C.c_void_p), ("prefix_stride", C.c_int64), ("suffix_len", C.c_void_p), ("suffix_pages", C.c_void_p),
                ("suffix_stride", C.c_int64), ("fold", C.c_void_p), ("out", C.c_void_p), ("out_stride", C.c_int64), ("site_m", C.c_int64),
                ("site_e", C.c_int64), ("out_codes", C.c_void_p), ("out_scales", C.c_void_p), ("row_status", C.c_void_p), ("reserved", C.c_uint64)]


class PickArgs(C.Structure):
    _fields_ = [("struct_size", C.c_uint32), ("rows", C.c_int32), ("vocab", C.c_int32), ("num_masks", C.c_int32), ("max_history", C.c_int32),
                ("max_bias", C.c_int32), ("reserved", C.c_uint32), ("logits", C.c_void_p),
                ("logits_stride", C.c_int64), ("params", C.c_void_p), ("history", C.c_void_p), ("history_stride", C.c_int64),
                ("history_len", C.c_void_p), ("bias_tokens", C.c_void_p), ("bias_values", C.c_void_p), ("bias_stride", C.c_int64),
                ("bias_len", C.c_void_p), ("masks", C.c_void_p), ("mask_stride", C.c_int64), ("mask_page", C.c_void_p), ("out_tokens", C.c_void_p),
                ("out_best", C.c_void_p), ("out_logits", C.c_void_p), ("out_stride", C.c_int64), ("row_status", C.c_void_p)]


class _ResidentCall:
    def __init__(self, lib: SslmLib, verb: str, args):
        self._fn = getattr(lib.dll, verb)
        self._fn.restype = C.c_int
        self._fn.argtypes = [C.c_void_p, C.c_void_p]
        self.verb, self.args, self._held, self._device = verb, args, [], None
        args.struct_size = C.sizeof(args)

    def _hold(self, name, t, dtype, shape, rows_strided=False):
        """The address of a tensor of this dtype and shape (None: any extent), dense but for the rows' stride."""
        if t is None:
            return None
        if str(t.dtype).split(".")[-1] != dtype:
            raise TypeError("%s: %s expected, got %s" % (name, dtype, t.dtype))
        if len(t.shape) != len(shape) or any(w is not None and g != w for g, w in zip(t.shape, shape)):
            raise ValueError("%s: shape %s expected, got %s" % (name, list(shape), list(t.shape)))
        if t.device.type != "cuda" or (self._device is not None and t.device != self._device):
            raise ValueError("%s: a tensor on %s expected, got one on %s" % (name, self._device or "a GPU", t.device))
        want = 1
        for i in range(len(shape) - 1, -1, -1):
            if rows_strided and i == 0:
                if t.shape[0] > 1 and t.stride(0) < want:
                    raise ValueError("%s: rows may not overlap" % name)
            elif t.shape[i] > 1 and t.stride(i) != want:
                raise ValueError("%s: dense elements expected, got strides %s" % (name, list(t.stride())))
            want *= t.shape[i]
        self._device = t.device
        self._held.append(t)
        return t.data_ptr()

    @staticmethod
    def _row_stride(t, width):
        return t.stride(0) if t is not None and t.shape[0] > 1 else width

    def run(self, stream=None):
        """Enqueues the call on `stream` (a cudaStream_t as an int; default: torch's current stream of the tensors' device)."""
        import torch
        if torch.cuda.current_device() != self._device.index:
            with torch.cuda.device(self._device):
                return self.run(stream)
        if stream is None:
            stream = torch.cuda.current_stream().cuda_stream
        st = self._fn(C.addressof(self.args), stream)
        if st != SSLM_OK:
            raise SslmError(self.verb, st)


class PrefixAttention(_ResidentCall):
    """sslm_b200_attention_prefix_resident. q int8 [rows, heads, head_dim] and out int32 of the same shape (rows may be
    strided), consts int64 [rows, kv_heads, 3], kv int8 [kv_heads, 2, pages, 16 * head_dim], group_start int32 [groups + 1],
    prefix_len int32 [groups], prefix_pages int32 [groups, n], suffix_len int32 [rows], suffix_pages int32 [rows, n], fold int32
    [heads, 3] or None; out_codes int8 [rows, heads * head_dim] and out_scales int64 [rows, 2] with site = (m, e); row_status int32 [rows].
    No length may exceed max_prefix / max_suffix (default: what the page tables hold)."""

    def __init__(self, lib, q, consts, kv, group_start, prefix_len, prefix_pages, suffix_len, suffix_pages, out, fold=None, max_prefix=None,
                 max_suffix=None, site=(0, 0), out_codes=None, out_scales=None, row_status=None):
        a = PrefixAttentionArgs()
        super().__init__(lib, "sslm_b200_attention_prefix_resident", a)
        rows, heads, hd = q.shape
        groups, kv_heads = prefix_len.shape[0], kv.shape[0]
        a.rows, a.groups, a.heads, a.kv_heads, a.head_dim = rows, groups, heads, kv_heads, hd
        a.q, a.q_stride = self._hold("q", q, "int8", (rows, heads, hd), True), self._row_stride(q, heads * hd)
        a.consts = self._hold("consts", consts, "int64", (rows, kv_heads, 3))
        a.kv, a.num_pages = self._hold("kv", kv, "int8", (kv_heads, 2, None, 16 * hd)), kv.shape[2]
        a.group_start = self._hold("group_start", group_start, "int32", (groups + 1,))
        a.prefix_len = self._hold("prefix_len", prefix_len, "int32", (groups,))
        a.prefix_pages = self._hold("prefix_pages", prefix_pages, "int32", (groups, None), True)
        a.prefix_stride = self._row_stride(prefix_pages, prefix_pages.shape[1])
        a.suffix_len = self._hold("suffix_len", suffix_len, "int32", (rows,))
        a.suffix_pages = self._hold("suffix_pages", suffix_pages, "int32", (rows, None), True)
        a.suffix_stride = self._row_stride(suffix_pages, suffix_pages.shape[1])
        a.max_prefix = min(32768, prefix_pages.shape[1] * 16) if max_prefix is None else max_prefix
        a.max_suffix = min(32768, suffix_pages.shape[1] * 16) if max_suffix is None else max_suffix
        if a.max_prefix > prefix_pages.shape[1] * 16 or a.max_suffix > suffix_pages.shape[1] * 16:
            raise ValueError("max_prefix / max_suffix: more than the page tables hold")
        a.fold = self._hold("fold", fold, "int32", (heads, 3))
        a.out, a.out_stride = self._hold("out", out, "int32", (rows, heads, hd), True), self._row_stride(out, heads * hd)
        a.site_m, a.site_e = site
        a.out_codes = self._hold("out_codes", out_codes, "int8", (rows, heads * hd))
        a.out_scales = self._hold("out_scales", out_scales, "int64", (rows, 2))
        a.row_status = self._hold("row_status", row_status, "int32", (rows,))


class Pick(_ResidentCall):
    """sslm_b200_pick_resident. logits int32 [rows, vocab] (rows may be strided), params int32 [rows, 3] (repetition in Q15, presence,
    frequency), history int32 [rows, n] with history_len int32 [rows], bias_tokens and bias_values int32 [rows, n] with bias_len int32
    [rows], masks uint8 [pages, ceil(vocab / 8)] with mask_page int32 [rows] (-1: none), out_tokens and out_best int32 [rows],
    out_logits int32 [rows, vocab] (may be `logits`), row_status int32 [rows]; what is None is left out."""

    def __init__(self, lib, logits, params=None, history=None, history_len=None, bias_tokens=None, bias_values=None, bias_len=None, masks=None,
                 mask_page=None, out_tokens=None, out_best=None, out_logits=None, row_status=None):
        a = PickArgs()
        super().__init__(lib, "sslm_b200_pick_resident", a)
        rows, vocab = logits.shape
        a.rows, a.vocab = rows, vocab
        a.logits, a.logits_stride = self._hold("logits", logits, "int32", (rows, vocab), True), self._row_stride(logits, vocab)
        a.params = self._hold("params", params, "int32", (rows, 3))
        if (history is None) != (history_len is None) or (masks is None) != (mask_page is None) or len({bias_tokens is None, bias_values is None, bias_len is None}) > 1:
            raise ValueError("a list comes with its lengths (and values), masks with mask_page")
        if history is not None:
            a.history, a.history_stride = self._hold("history", history, "int32", (rows, None), True), self._row_stride(history, history.shape[1])
            a.max_history = history.shape[1]
            a.history_len = self._hold("history_len", history_len, "int32", (rows,))
        if bias_tokens is not None:
            a.bias_tokens = self._hold("bias_tokens", bias_tokens, "int32", (rows, None))
            a.bias_values = self._hold("bias_values", bias_values, "int32", tuple(bias_tokens.shape))
            a.bias_stride = a.max_bias = bias_tokens.shape[1]
            a.bias_len = self._hold("bias_len", bias_len, "int32", (rows,))
        if masks is not None:
            a.masks, a.num_masks = self._hold("masks", masks, "uint8", (None, None), True), masks.shape[0]
            if masks.shape[1] < (vocab + 7) // 8:
                raise ValueError("masks: %d bytes a page expected, got %d" % ((vocab + 7) // 8, masks.shape[1]))
            a.mask_stride = self._row_stride(masks, masks.shape[1])
            a.mask_page = self._hold("mask_page", mask_page, "int32", (rows,))
        a.out_tokens = self._hold("out_tokens", out_tokens, "int32", (rows,))
        a.out_best = self._hold("out_best", out_best, "int32", (rows,))
        a.out_logits = self._hold("out_logits", out_logits, "int32", (rows, vocab), True)
        a.out_stride = self._row_stride(out_logits, vocab)
        a.row_status = self._hold("row_status", row_status, "int32", (rows,))


def parse_save_blob(blob: bytes, hidden_size: int) -> dict:
    """Fields of an SSB3 sequence blob (src/sslm_abi.cpp:2620-2716)."""
    assert blob[0:4] == b"SSB3"
    ctx_len, layer_index, cur_tok, hm, he, sat = struct.unpack_from("<qIiqqQ", blob, 60)
    off = 120
    residual = b""
    if layer_index != 0:
        residual = blob[off:off + hidden_size]
        off += hidden_size
    hist = struct.unpack_from("<Q", blob, 112)[0]
    off += 4 * hist
    nblk = struct.unpack_from("<I", blob, off)[0]
    off += 4
    return {"context_length": ctx_len, "layer_index": layer_index, "current_token": cur_tok,
            "hidden_scale": (hm, he), "kv_saturation_count": sat, "residual": residual,
            "kv_block_count": nblk, "kv": blob[off:]}
