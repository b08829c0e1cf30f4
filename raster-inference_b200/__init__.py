"""B200-native deterministic integer-weight transformer path (rdet).

Host-side mirror of casettek/raster-inference's det routine API over the
C ABI in ``include/rdet.h`` (``librdet.so`` in this directory).  The names
follow the reference routines:

    load_transformer_state_model_from_det_num_wgt_path   io.rs:1043
    input_embedding                                      routines/input_embedding/mod.rs:17
    run_prefill (prefill_layer routine family)            executors/native.rs:153
    select_output_token                                  decode_select_token/native/tiles.rs:22
    decode_transition                                    executors/native.rs:339-437
    run_output_decode                                    executors/native.rs:265

There is no CPU fallback: every entry point raises ImportError when the CUDA
library is missing, and fails with ``RdetError`` carrying the reference's
error message when the C ABI reports a failure.
"""
from __future__ import annotations

import ctypes as C
import json
import os

import numpy as np

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "librdet.so")

RDET_OK, RDET_NONE = 0, 1
BUF_EMBEDDING, BUF_HIDDEN, BUF_LOGITS, BUF_LAYER_OUTPUT, BUF_KV, BUF_KV_K, BUF_KV_V = range(7)
FLAG_LAYER_COMMITMENTS = 1
FLAG_NO_TENSOR_CORES = 2

# Exported symbols, in the order include/rdet.h declares them.
SYMBOLS = [
    "rdet_open", "rdet_open_synthetic", "rdet_close", "rdet_get_model_info", "rdet_seq_new", "rdet_seq_free",
    "rdet_seq_position", "rdet_embed", "rdet_prefill", "rdet_prefill_begin", "rdet_prefill_range",
    "rdet_prefill_finalize", "rdet_select", "rdet_select_batch", "rdet_decode", "rdet_decode_begin", "rdet_decode_range",
    "rdet_decode_finalize", "rdet_generate", "rdet_select_rules", "rdet_tree_decode", "rdet_tree_select",
    "rdet_tree_accept", "rdet_read", "rdet_commitment", "rdet_kv_prefix_commitments",
    "rdet_det_gemv", "rdet_det_linear",
    "rdet_det_attention_decode", "rdet_det_attention_decode_noalloc", "rdet_det_attention_prefill", "rdet_convert_to_wgt",
    "rdet_det_attention_tree_workspace", "rdet_det_attention_tree", "rdet_det_logits_rules", "rdet_det_tree_commit", "rdet_det_status",
    "rdet_get_stream", "rdet_tensor_core_prefill", "rdet_nccl_unique_id", "rdet_tp_init", "rdet_tp_world", "rdet_tp_shard_logits", "rdet_tp_ipc_export", "rdet_tp_ipc_connect", "rdet_seq_kernels_per_step", "rdet_last_error",
    "rdet_version",
]


NO_TOKEN = 0xFFFFFFFF
MAX_TREE_NODES = 64


class RdetError(RuntimeError):
    def __init__(self, code: int, msg: str):
        super().__init__(f"rdet error {code}: {msg}")
        self.code = code
        self.msg = msg


class Opts(C.Structure):
    _fields_ = [("device", C.c_int32), ("max_prefill", C.c_uint32), ("flags", C.c_uint32)]


class ModelInfo(C.Structure):
    _fields_ = [("hidden_size", C.c_uint32), ("vocab_size", C.c_uint32), ("num_layers", C.c_uint32),
                ("num_heads", C.c_uint32), ("ple_dim", C.c_uint32), ("intermediate_size", C.c_uint32),
                ("weight_bytes", C.c_uint64)]


class TreeSeq(C.Structure):
    _fields_ = [("k_cache", C.c_void_p), ("v_cache", C.c_void_p), ("k_tree", C.c_void_p), ("v_tree", C.c_void_p),
                ("parents", C.c_void_p), ("cap", C.c_uint32), ("context", C.c_uint32), ("tree_cap", C.c_uint32),
                ("n_nodes", C.c_uint32)]


class LogitRow(C.Structure):
    _fields_ = [("logits", C.c_void_p), ("out", C.c_void_p), ("allow", C.c_void_p), ("history", C.c_void_p),
                ("bias_ids", C.c_void_p), ("bias_values", C.c_void_p), ("history_len", C.c_uint32),
                ("n_bias", C.c_uint32), ("repetition", C.c_int32), ("frequency", C.c_int32),
                ("presence", C.c_int32), ("parent", C.c_int32), ("token", C.c_uint32)]


class Rules(C.Structure):
    """Rules of one sequence's selection (rdet_rules); pointers are host memory."""
    _fields_ = [("allow", C.c_void_p), ("history", C.c_void_p), ("bias_ids", C.c_void_p),
                ("bias_values", C.c_void_p), ("history_len", C.c_uint32), ("n_bias", C.c_uint32),
                ("repetition", C.c_int32), ("frequency", C.c_int32), ("presence", C.c_int32)]


class TreeMove(C.Structure):
    _fields_ = [("cache", C.c_void_p), ("draft", C.c_void_p), ("cap", C.c_uint32), ("draft_cap", C.c_uint32),
                ("kv_heads", C.c_uint32), ("head_dim", C.c_uint32), ("context", C.c_uint32), ("path", C.c_uint32)]


_lib = None


def lib() -> C.CDLL:
    """Load librdet.so (raises if it was not built — there is no fallback)."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise ImportError(f"{LIB_PATH} is missing: build it with `make -C {_HERE}` (no CPU fallback exists)")
    L = C.CDLL(LIB_PATH)
    p, i32, u32, u64, sz = C.c_void_p, C.c_int32, C.c_uint32, C.c_uint64, C.c_size_t
    sig = {
        "rdet_open": [C.c_char_p, p, p],
        "rdet_open_synthetic": [C.c_char_p, u64, i32, p, p],
        "rdet_close": [p],
        "rdet_get_model_info": [p, p],
        "rdet_seq_new": [p, u32, p],
        "rdet_seq_free": [p],
        "rdet_seq_position": [p, p],
        "rdet_embed": [p, p, sz, p],
        "rdet_prefill": [p, p, p, sz],
        "rdet_prefill_begin": [p, p, p, sz],
        "rdet_prefill_range": [p, p, u32, u32],
        "rdet_prefill_finalize": [p, p],
        "rdet_select": [p, p, p],
        "rdet_select_batch": [p, p, sz, p],
        "rdet_tp_shard_logits": [p, i32],
        "rdet_decode": [p, p, p, sz],
        "rdet_decode_begin": [p, p, u32],
        "rdet_decode_range": [p, p, u32, u32],
        "rdet_decode_finalize": [p, p],
        "rdet_generate": [p, p, u32, p],
        "rdet_select_rules": [p, p, sz, p, p],
        "rdet_tree_decode": [p, p, sz, p, p, p],
        "rdet_tree_select": [p, p, sz, p, p],
        "rdet_tree_accept": [p, p, sz, p, p],
        "rdet_read": [p, p, i32, i32, i32, p, sz, p],
        "rdet_commitment": [p, p, i32, i32, C.c_char_p],
        "rdet_kv_prefix_commitments": [p, p, C.c_uint32, C.c_char_p],
        "rdet_det_gemv": [p, p, i32, u32, u32, p, p],
        "rdet_det_linear": [p, u32, p, i32, u32, u32, p, p],
        "rdet_det_attention_decode": [p, p, p, u32, u32, u32, u32, u32, u32, p, p],
        "rdet_det_attention_decode_noalloc": [p, p, p, u32, u32, u32, u32, u32, u32, p, p],
        "rdet_det_attention_prefill": [p, p, p, u32, u32, u32, u32, u32, u32, u32, p, p],
        "rdet_convert_to_wgt": [p, i32, C.c_uint64, C.c_uint64, p, p, p, p],
        "rdet_det_attention_tree_workspace": [p, u32, u32, u32, u32, u32, p],
        "rdet_det_attention_tree": [p, u32, p, u32, u32, u32, u32, p, p, sz, p],
        "rdet_det_logits_rules": [p, u32, u32, p, p],
        "rdet_det_tree_commit": [p, u32, p, p, u32, p],
        "rdet_det_status": [p],
        "rdet_get_stream": [p, p],
        "rdet_tensor_core_prefill": [p],
        "rdet_nccl_unique_id": [p, sz],
        "rdet_tp_init": [p, i32, i32, p, sz],
        "rdet_tp_world": [p],
        "rdet_tp_ipc_export": [p, u32, p, sz, p],
        "rdet_tp_ipc_connect": [p, p, sz, i32],
        "rdet_seq_kernels_per_step": [p, p],
        "rdet_last_error": [C.c_char_p, sz],
    }
    for name, args in sig.items():
        f = getattr(L, name)
        f.argtypes = args
        f.restype = i32
    L.rdet_version.restype = C.c_char_p
    L.rdet_version.argtypes = []
    _lib = L
    return L


def _check(rc: int):
    if rc < 0:
        buf = C.create_string_buffer(4096)
        lib().rdet_last_error(buf, 4096)
        raise RdetError(rc, buf.value.decode(errors="replace"))
    return rc


def _ptr(a: np.ndarray):
    return a.ctypes.data_as(C.c_void_p)


class Model:
    """Gemma-4 det model resident in HBM (Gemma4TransformerModel, model/gemma/transformer.rs:560)."""

    def __init__(self, handle, config: dict | None):
        self._h = handle
        self.config = config
        info = ModelInfo()
        _check(lib().rdet_get_model_info(self._h, C.byref(info)))
        self.H, self.V, self.L = info.hidden_size, info.vocab_size, info.num_layers
        self.Hq, self.P, self.F = info.num_heads, info.ple_dim, info.intermediate_size
        self.weight_bytes = info.weight_bytes
        self.max_prefill = 4096

    @classmethod
    def open(cls, model_dir: str, device: int = 0, max_prefill: int = 0, layer_commitments: bool = False,
             tensor_cores: bool = True):
        flags = (FLAG_LAYER_COMMITMENTS if layer_commitments else 0) | (0 if tensor_cores else FLAG_NO_TENSOR_CORES)
        opts = Opts(device, max_prefill, flags)
        h = C.c_void_p()
        _check(lib().rdet_open(model_dir.encode(), C.byref(opts), C.byref(h)))
        with open(os.path.join(model_dir, "config.json")) as f:
            cfg = json.load(f)
        model = cls(h, cfg)
        model.max_prefill = max_prefill or model.max_prefill
        return model

    @classmethod
    def synthetic(cls, config: dict, seed: int, width: int = 16, device: int = 0, max_prefill: int = 0,
                  layer_commitments: bool = False, tensor_cores: bool = True):
        flags = (FLAG_LAYER_COMMITMENTS if layer_commitments else 0) | (0 if tensor_cores else FLAG_NO_TENSOR_CORES)
        opts = Opts(device, max_prefill, flags)
        h = C.c_void_p()
        _check(lib().rdet_open_synthetic(json.dumps(config).encode(), seed, width, C.byref(opts), C.byref(h)))
        model = cls(h, config)
        model.max_prefill = max_prefill or model.max_prefill
        return model

    def close(self):
        if getattr(self, "_h", None):
            lib().rdet_close(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def tp_init(self, rank: int, world: int, uid: bytes):
        """Shard the batched decode over `world` ranks (rdet_tp_init); every rank
        opened the same model and passes the same id from nccl_unique_id()."""
        buf = C.create_string_buffer(bytes(uid), len(uid))
        _check(lib().rdet_tp_init(self._h, rank, world, buf, len(uid)))

    def tp_shard_logits(self, on: bool = True) -> None:
        """Vocab-sharded selection (rdet_tp_shard_logits): batched decodes end
        with a global argmax over (value, index) pairs instead of gathering
        the logit rows; take the tokens with select_batch."""
        _check(lib().rdet_tp_shard_logits(self._h, 1 if on else 0))

    def tp_ipc_export(self, max_batch: int) -> bytes:
        """This rank's NVLink reduction buffers for batches of up to max_batch
        sequences (rdet_tp_ipc_export): an opaque blob for every other rank."""
        buf = C.create_string_buffer(256)
        n = C.c_size_t(0)
        _check(lib().rdet_tp_ipc_export(self._h, max_batch, buf, 256, C.byref(n)))
        return buf.raw[: n.value]

    def tp_ipc_connect(self, blobs) -> None:
        """Map the other ranks' reduction buffers (all ranks' export blobs in
        rank order, rdet_tp_ipc_connect): the sharded decode then reduces over
        NVLink instead of NCCL."""
        each = len(blobs[0])
        assert all(len(b) == each for b in blobs)
        buf = C.create_string_buffer(b"".join(blobs), each * len(blobs))
        _check(lib().rdet_tp_ipc_connect(self._h, buf, each, len(blobs)))

    @property
    def tp_world(self) -> int:
        return int(lib().rdet_tp_world(self._h))

    @property
    def tensor_core_prefill(self) -> bool:
        """Whether prefill linears of >= 32 tokens run on the tcgen05 tensor cores."""
        return bool(lib().rdet_tensor_core_prefill(self._h))

    @property
    def stream(self) -> int:
        """cudaStream_t (as an int) on which this model launches its work."""
        v = C.c_void_p()
        _check(lib().rdet_get_stream(self._h, C.byref(v)))
        return v.value or 0

    def new_sequence(self, max_ctx: int) -> "Sequence":
        h = C.c_void_p()
        _check(lib().rdet_seq_new(self._h, max_ctx, C.byref(h)))
        seq = Sequence(self, h)
        seq.max_ctx = max_ctx
        return seq

    def embed(self, ids) -> np.ndarray:
        ids = np.ascontiguousarray(ids, dtype=np.uint32)
        out = np.zeros((ids.size, self.H), dtype=np.int32)
        _check(lib().rdet_embed(self._h, _ptr(ids), ids.size, _ptr(out)))
        return out


class Sequence:
    """One sequence's decode state (TransformerDecodeState) with its KV cache in HBM."""

    def __init__(self, model: Model, handle):
        self.model = model
        self._h = handle

    def free(self):
        if getattr(self, "_h", None):
            if getattr(self.model, "_h", None):  # closing the model already freed it
                lib().rdet_seq_free(self._h)
            self._h = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass

    @property
    def position(self) -> int:
        v = C.c_uint32()
        _check(lib().rdet_seq_position(self._h, C.byref(v)))
        return v.value

    # -- routines -------------------------------------------------------------
    def prefill(self, ids):
        ids = np.ascontiguousarray(ids, dtype=np.uint32)
        _check(lib().rdet_prefill(self.model._h, self._h, _ptr(ids), ids.size))

    def prefill_begin(self, ids):
        ids = np.ascontiguousarray(ids, dtype=np.uint32)
        _check(lib().rdet_prefill_begin(self.model._h, self._h, _ptr(ids), ids.size))

    def prefill_range(self, start: int, end: int):
        _check(lib().rdet_prefill_range(self.model._h, self._h, start, end))

    def prefill_finalize(self):
        _check(lib().rdet_prefill_finalize(self.model._h, self._h))

    def select(self) -> int:
        t = C.c_uint32()
        _check(lib().rdet_select(self.model._h, self._h, C.byref(t)))
        return t.value

    def decode(self, token: int):
        arr = (C.c_void_p * 1)(self._h)
        toks = np.array([token], dtype=np.uint32)
        _check(lib().rdet_decode(self.model._h, arr, _ptr(toks), 1))

    def decode_begin(self, token: int):
        _check(lib().rdet_decode_begin(self.model._h, self._h, token))

    def decode_range(self, start: int, end: int):
        _check(lib().rdet_decode_range(self.model._h, self._h, start, end))

    def decode_finalize(self):
        _check(lib().rdet_decode_finalize(self.model._h, self._h))

    def generate(self, n: int) -> list[int]:
        out = np.zeros(max(n, 1), dtype=np.uint32)
        _check(lib().rdet_generate(self.model._h, self._h, n, _ptr(out)))
        return [int(v) for v in out[:n]]

    def kernels_per_step(self) -> int:
        v = C.c_uint32()
        _check(lib().rdet_seq_kernels_per_step(self._h, C.byref(v)))
        return v.value

    # -- canonical bytes / commitments -------------------------------------------
    def read(self, which: int, layer: int = 0, arg: int = 0) -> np.ndarray:
        size = C.c_size_t()
        _check(lib().rdet_read(self.model._h, self._h, which, layer, arg, None, 0, C.byref(size)))
        out = np.zeros(size.value // 4, dtype=np.int32)
        _check(lib().rdet_read(self.model._h, self._h, which, layer, arg, _ptr(out), size.value, C.byref(size)))
        return out

    def commitment(self, which: int, layer: int = 0):
        buf = C.create_string_buffer(65)
        rc = _check(lib().rdet_commitment(self.model._h, self._h, which, layer, buf))
        return None if rc == RDET_NONE else buf.value.decode()

    def kv_prefix_commitments(self, n: int) -> list:
        """commitment(BUF_KV, p) for p = 1..n in one call (None where a
        prefix holds a KV-sharing layer)."""
        buf = C.create_string_buffer(65 * max(n, 1))
        _check(lib().rdet_kv_prefix_commitments(self.model._h, self._h, n, buf))
        out = []
        for p in range(n):
            h = buf.raw[65 * p:65 * p + 64]
            out.append(None if h[0] == 0 else h.decode())
        return out

    def logits(self) -> np.ndarray:
        return self.read(BUF_LOGITS)


def nccl_unique_id() -> bytes:
    """A fresh NCCL id (128 bytes) for Model.tp_init on every rank."""
    buf = C.create_string_buffer(128)
    _check(lib().rdet_nccl_unique_id(buf, 128))
    return buf.raw


def decode_batch(model: Model, seqs, tokens):
    """decode_transition over a ragged batch (one token per sequence)."""
    arr = (C.c_void_p * len(seqs))(*[s._h for s in seqs])
    toks = np.ascontiguousarray(tokens, dtype=np.uint32)
    _check(lib().rdet_decode(model._h, arr, _ptr(toks), len(seqs)))


def select_batch(model: Model, seqs) -> list[int]:
    """select_output_token for every sequence in one launch (argmax_first of
    each sequence's logits; after a vocab-sharded tensor-parallel decode,
    the tokens its global argmax selected)."""
    n = len(seqs)
    arr = (C.c_void_p * max(n, 1))(*[s._h for s in seqs])
    out = np.zeros(max(n, 1), dtype=np.uint32)
    _check(lib().rdet_select_batch(model._h, arr, n, _ptr(out)))
    return [int(v) for v in out[:n]]


# ---- drafted decoding ----------------------------------------------------------------
def _handles(seqs):
    return (C.c_void_p * max(len(seqs), 1))(*[s._h for s in seqs])


def _rules(model, rules, masks):
    """rdet_rules array from one dict per sequence (masks[i]: the allow masks
    of sequence i), or None: allow (u32 words,
    for tree_select one row per node), history (token ids), bias ({token id:
    Q16.16 value}), repetition, frequency and presence (Q16.16); what a dict
    leaves out is no rule of that kind.  The array keeps the memory it names."""
    if rules is None:
        return None
    if len(rules) != len(masks):
        raise ValueError("one dict of rules per sequence")
    out = (Rules * max(len(rules), 1))()
    out.keep = []
    for o, r, n in zip(out, rules, masks):
        unknown = set(r) - {"allow", "history", "bias", "repetition", "frequency", "presence"}
        if unknown:
            raise TypeError(f"unknown rules {sorted(unknown)}")
        hist = np.ascontiguousarray(r.get("history", ()), dtype=np.uint32)
        bias = r.get("bias", {})
        ids = np.array(list(bias.keys()), dtype=np.uint32)
        vals = np.array(list(bias.values()), dtype=np.int32)
        if hist.ndim != 1:
            raise ValueError("history: a list of token ids")
        out.keep += [hist, ids, vals]
        if r.get("allow") is not None:
            allow = np.ascontiguousarray(r["allow"], dtype=np.uint32)
            if allow.size != n * ((model.V + 31) // 32):
                raise ValueError(f"allow: {n} masks of {(model.V + 31) // 32} words")
            out.keep.append(allow)
            o.allow = allow.ctypes.data
        o.history, o.history_len = hist.ctypes.data, hist.size
        o.bias_ids, o.bias_values, o.n_bias = ids.ctypes.data, vals.ctypes.data, ids.size
        o.repetition = r.get("repetition", 1 << 16)
        o.frequency, o.presence = r.get("frequency", 0), r.get("presence", 0)
    return out


def select_rules(model: Model, seqs, rules) -> list[int]:
    """The greedy token of each sequence under its rules (rdet_select_rules);
    NO_TOKEN where the mask allows none."""
    out = np.zeros(max(len(seqs), 1), dtype=np.uint32)
    _check(lib().rdet_select_rules(model._h, _handles(seqs), len(seqs), _rules(model, rules, [1] * len(seqs)), _ptr(out)))
    return [int(v) for v in out[:len(seqs)]]


def tree_decode(model: Model, seqs, tokens, parents):
    """Every node of each sequence's drafted tree in one pass (rdet_tree_decode):
    tokens[i] and parents[i] list sequence i's nodes."""
    counts = np.array([len(t) for t in tokens], dtype=np.uint32)
    if any(len(t) != len(q) for t, q in zip(tokens, parents)) or not len(seqs) == len(tokens) == len(parents):
        raise ValueError("one list of tokens and one of parents per sequence, of the same length")
    toks = np.array([t for row in tokens for t in row], dtype=np.uint32)
    par = np.array([q for row in parents for q in row], dtype=np.int32)
    _check(lib().rdet_tree_decode(model._h, _handles(seqs), len(seqs), _ptr(counts), _ptr(toks), _ptr(par)))
    for s, t in zip(seqs, tokens):
        s._tree = len(t)


def tree_select(model: Model, seqs, rules=None) -> list[list[int]]:
    """The greedy token after every node of each sequence's drafted tree
    (rdet_tree_select), under rules when given."""
    n = [getattr(s, "_tree", 0) for s in seqs]
    out = np.zeros(max(sum(n), 1), dtype=np.uint32)
    _check(lib().rdet_tree_select(model._h, _handles(seqs), len(seqs), _rules(model, rules, n), _ptr(out)))
    at = np.cumsum([0] + n)
    return [[int(v) for v in out[a:b]] for a, b in zip(at[:-1], at[1:])]


def tree_accept(model: Model, seqs, paths):
    """Commits one path of each sequence's drafted tree (rdet_tree_accept)."""
    if len(paths) != len(seqs):
        raise ValueError("one path per sequence")
    counts = np.array([len(p) for p in paths], dtype=np.uint32)
    nodes = np.array([n for p in paths for n in p] + [0], dtype=np.uint32)
    _check(lib().rdet_tree_accept(model._h, _handles(seqs), len(seqs), _ptr(counts), _ptr(nodes)))


# ---- reference-named entry points ---------------------------------------------------
def load_transformer_state_model_from_det_num_wgt_path(model_dir: str, **kw) -> Model:
    return Model.open(model_dir, **kw)


def input_embedding(model: Model, prompt_token_ids) -> np.ndarray:
    return model.embed(prompt_token_ids)


def run_prefill(model: Model, prompt_token_ids, max_ctx: int) -> Sequence:
    seq = model.new_sequence(max_ctx)
    seq.prefill(prompt_token_ids)
    return seq


def select_output_token(seq: Sequence) -> int:
    return seq.select()


def decode_transition(seq: Sequence, next_token: int):
    seq.decode(next_token)


def run_output_decode(seq: Sequence, max_new_tokens: int) -> list[int]:
    """Greedy loop of executors/native.rs:265-450 (select, then decode)."""
    return seq.generate(max_new_tokens)


def det_gemv(x_ptr: int, w_ptr: int, width: int, rows: int, cols: int, y_ptr: int, stream: int = 0):
    """GEMV on caller-owned device pointers (integers, e.g. torch data_ptr())."""
    _check(lib().rdet_det_gemv(C.c_void_p(x_ptr), C.c_void_p(w_ptr), width, rows, cols, C.c_void_p(y_ptr),
                               C.c_void_p(stream) if stream else None))


def det_linear(x_ptr: int, s: int, w_ptr: int, width: int, rows: int, cols: int, y_ptr: int, stream: int = 0):
    _check(lib().rdet_det_linear(C.c_void_p(x_ptr), s, C.c_void_p(w_ptr), width, rows, cols, C.c_void_p(y_ptr),
                                 C.c_void_p(stream) if stream else None))


def det_attention_decode(q_ptr: int, k_ptr: int, v_ptr: int, cap: int, num_heads: int, num_kv_heads: int,
                         head_dim: int, position: int, window: int, out_ptr: int, stream: int = 0):
    """Decode attention of one token on caller-owned device memory (rdet_det_attention_decode)."""
    _check(lib().rdet_det_attention_decode(C.c_void_p(q_ptr), C.c_void_p(k_ptr), C.c_void_p(v_ptr), cap, num_heads,
                                           num_kv_heads, head_dim, position, window, C.c_void_p(out_ptr),
                                           C.c_void_p(stream) if stream else None))


def det_attention_prefill(q_ptr: int, k_ptr: int, v_ptr: int, cap: int, n_tokens: int, num_heads: int,
                          num_kv_heads: int, head_dim: int, window: int, out_ptr: int, tensor_cores: bool = True,
                          stream: int = 0):
    """Prefill attention of a prompt on caller-owned device memory
    (rdet_det_attention_prefill); tensor_cores=False forces the CUDA-core kernel."""
    _check(lib().rdet_det_attention_prefill(C.c_void_p(q_ptr), C.c_void_p(k_ptr), C.c_void_p(v_ptr), cap, n_tokens,
                                            num_heads, num_kv_heads, head_dim, window,
                                            0 if tensor_cores else FLAG_NO_TENSOR_CORES, C.c_void_p(out_ptr),
                                            C.c_void_p(stream) if stream else None))


SRC_DTYPES = {"F32": 0, "BF16": 1, "F16": 2}


def convert_to_wgt(src_ptr: int, dtype: str, rows: int, row_len: int, out_ptr: int, row_mass_ptr: int,
                   stats_ptr: int, stream: int = 0):
    """safetensors values -> Q16.16 weights on the GPU (rdet_convert_to_wgt):
    out = f32_to_wgt(value), row_mass = sum |out| per row, stats = [non-finite
    count, does not fit i16]; all device pointers."""
    _check(lib().rdet_convert_to_wgt(C.c_void_p(src_ptr), SRC_DTYPES[dtype], rows, row_len, C.c_void_p(out_ptr),
                                     C.c_void_p(row_mass_ptr), C.c_void_p(stats_ptr),
                                     C.c_void_p(stream) if stream else None))


def det_attention_decode_noalloc(q_ptr: int, k_ptr: int, v_ptr: int, cap: int, num_heads: int, num_kv_heads: int,
                                 head_dim: int, position: int, window: int, out_ptr: int, stream: int = 0):
    """rdet_det_attention_decode without any device allocation, for callers
    that cannot allocate device memory while they run (all of HBM handed to
    weights and KV caches up front, or a fixed per-step footprint).  Scratch
    is the library's fixed 4.8 MiB array; limits: 16 heads, head_dim 512,
    4096 attended rows.  Calls that overlap on the GPU race on that array."""
    _check(lib().rdet_det_attention_decode_noalloc(C.c_void_p(q_ptr), C.c_void_p(k_ptr), C.c_void_p(v_ptr), cap,
                                                   num_heads, num_kv_heads, head_dim, position, window,
                                                   C.c_void_p(out_ptr), C.c_void_p(stream) if stream else None))


# ---- verification of drafted tokens ---------------------------------------------------
class Descriptors:
    """A host descriptor array of the draft-verification operators with the
    host memory it points into; device pointers stay the caller's."""

    def __init__(self, ctype, items, keep=()):
        self.n = len(items)
        self.array = (ctype * max(self.n, 1))(*[ctype(**it) for it in items])
        self.keep = keep


def tree_seqs(seqs) -> Descriptors:
    """rdet_tree_seq array from dicts of k_cache, v_cache, cap, context,
    k_tree, v_tree, tree_cap (device pointers as integers) and parents (list)."""
    keep, items = [], []
    for s in seqs:
        par = np.ascontiguousarray(s["parents"], dtype=np.int32)
        keep.append(par)
        items.append({**s, "parents": par.ctypes.data, "n_nodes": par.size})
    return Descriptors(TreeSeq, items, keep)


def det_attention_tree_workspace(seqs: Descriptors, num_heads: int, num_kv_heads: int, head_dim: int,
                                 window: int) -> int:
    """Bytes of device workspace that det_attention_tree needs for these trees."""
    n = C.c_size_t(0)
    _check(lib().rdet_det_attention_tree_workspace(seqs.array, seqs.n, num_heads, num_kv_heads, head_dim, window,
                                                   C.byref(n)))
    return n.value


def det_attention_tree(seqs: Descriptors, q_ptr: int, num_heads: int, num_kv_heads: int, head_dim: int, window: int,
                       out_ptr: int, ws_ptr: int, ws_bytes: int, stream: int = 0):
    """Attention of every node of a tree of drafted tokens over its sequence's
    cache rows, its ancestors and itself (rdet_det_attention_tree)."""
    _check(lib().rdet_det_attention_tree(seqs.array, seqs.n, q_ptr, num_heads, num_kv_heads, head_dim, window,
                                         out_ptr, ws_ptr, ws_bytes, stream))


def logit_rows(rows) -> Descriptors:
    """rdet_logit_row array from dicts; every field but `logits` may be left
    out (no rule of that kind)."""
    base = {"repetition": 1 << 16, "parent": -1, "token": NO_TOKEN}
    return Descriptors(LogitRow, [{**base, **r} for r in rows])


def det_logits_rules(rows: Descriptors, vocab: int, tokens_ptr: int, stream: int = 0):
    """Penalties, biases and the mask of allowed tokens on logits rows, and the
    greedy token of each (rdet_det_logits_rules)."""
    _check(lib().rdet_det_logits_rules(rows.array, rows.n, vocab, tokens_ptr, stream))


def tree_moves(moves, paths) -> Descriptors:
    """rdet_tree_move array from dicts of cache, draft, cap, draft_cap,
    kv_heads, head_dim, context and path (an index into `paths`, lists of nodes)."""
    nodes = np.ascontiguousarray([n for p in paths for n in p], dtype=np.uint32)
    off = np.ascontiguousarray(np.cumsum([0] + [len(p) for p in paths]), dtype=np.uint32)
    d = Descriptors(TreeMove, list(moves), (nodes, off))
    d.nodes, d.path_off, d.n_paths = nodes.ctypes.data, off.ctypes.data, len(paths)
    return d


def det_tree_commit(moves: Descriptors, stream: int = 0):
    """The drafted K/V rows of accepted paths into the caches (rdet_det_tree_commit)."""
    _check(lib().rdet_det_tree_commit(moves.array, moves.n, moves.nodes, moves.path_off, moves.n_paths, stream))


def det_status(stream: int = 0):
    """Waits for the stream and raises when a kernel on the current device gave
    up on a pipeline wait since this was last asked (rdet_det_status)."""
    _check(lib().rdet_det_status(stream))
