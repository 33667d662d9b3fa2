"""ctypes binding of libgpt2_b200.so (the C ABI declared in include/gpt2_b200.h).

This is plumbing for the tests and bench.py: it loads the in-tree shared library, declares every
entry point's signature, and offers thin helpers that pass torch tensors' device pointers. All work
happens in the CUDA kernels behind the C ABI; if the library is missing, loading raises instead of
falling back to anything else.
"""
from __future__ import annotations

import ctypes
import os
import re

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
LIB_PATH = os.path.join(HERE, "lib", "libgpt2_b200.so")
HEADER = os.path.join(ROOT, "include", "gpt2_b200.h")

OK, EINVAL, ECUDA, ENOMEM, EDEVICE, ETIMEOUT, ECAPTURE = range(7)

# Device status bits (bare-metal-gpt2_b200/csrc/common.cuh).
ST_PREFILL_LOAD_TIMEOUT = 1 << 0
ST_PREFILL_MMA_TIMEOUT = 1 << 1
ST_PREFILL_SOFTMAX_TIMEOUT = 1 << 2
ST_PREFILL_SMEM_ALIGN = 1 << 3
ST_PREFILL_DRAIN_TIMEOUT = 1 << 4
ST_DECODE_BAD_LEN = 1 << 8
ST_KV_BAD_POS = 1 << 9
ST_DECODE_TIMEOUT = 1 << 10
ST_LINEAR_TIMEOUT = 1 << 11
ST_MODEL_BAD_TOKEN = 1 << 12
ST_KV8_BAD_LEN = 1 << 13
ST_KV8_BAD_PAGE = 1 << 14
ST_KV8_NO_PAGE = 1 << 15
ST_TEST_WAIT_TIMEOUT = 1 << 16
ST_KV8_NONFINITE = 1 << 17
ST_KV8_BAD_PARENT = 1 << 18
ST_BEAM_LOGIT = 1 << 19
ST_W4_NONFINITE = 1 << 20
ST_EDIT_BAD_INPUT = 1 << 21
ST_EDIT_NO_TOKEN = 1 << 22

LINEAR_STORE, LINEAR_GELU, LINEAR_RESID = 0, 1, 2
GEN_ATTENTION_ONLY = 1
KV8_KINDS = {"int8": 0, "e4m3": 1}
BEAM_HALF, BEAM_FLOAT = 0, 1

# GPT-2-124M (the reference's model/config.h).
N_LAYER, N_HEAD, N_EMBD, VOCAB, N_CTX = 12, 12, 768, 50257, 1024
FFN, QKV_DIM = 4 * N_EMBD, 3 * N_EMBD
# Per-layer tensors in GPT2LayerGPU order (cuda/kernels.cuh:19-23) with their shapes.
LAYER_TENSORS = (
    ("ln1_g", (N_EMBD,)), ("ln1_b", (N_EMBD,)), ("qkv_w", (QKV_DIM, N_EMBD)), ("qkv_b", (QKV_DIM,)),
    ("attn_proj_w", (N_EMBD, N_EMBD)), ("attn_proj_b", (N_EMBD,)), ("ln2_g", (N_EMBD,)),
    ("ln2_b", (N_EMBD,)), ("fc_w", (FFN, N_EMBD)), ("fc_b", (FFN,)), ("proj_w", (N_EMBD, FFN)),
    ("proj_b", (N_EMBD,)),
)


class GPT2KVCache(ctypes.Structure):
    """Same layout as GPT2KVCache in the reference's cuda/kvcache.cuh:39-44."""

    _fields_ = [
        ("data", ctypes.c_void_p),
        ("bytes", ctypes.c_size_t),
        ("maxT", ctypes.c_int),
        ("nLayer", ctypes.c_int),
        ("nHead", ctypes.c_int),
        ("headDim", ctypes.c_int),
        ("len", ctypes.c_int),
    ]


class GPT2Backend(ctypes.Structure):
    """Same layout as GPT2Backend in the reference's cuda/kernels.cuh:68-86."""

    _fields_ = [("name", ctypes.c_char_p)] + [
        (n, ctypes.c_void_p)
        for n in ("embed", "layernorm", "matmul", "attention", "gelu", "add", "matmul_q", "gemv",
                  "gemv_q")
    ]


class GPT2KV8Cache(ctypes.Structure):
    """The paged 8-bit cache descriptor of include/gpt2_b200.h."""

    _fields_ = [(n, ctypes.c_void_p) for n in ("data", "scale", "ref", "table", "len", "work")] + [
        ("work_bytes", ctypes.c_size_t)] + [
        (n, ctypes.c_int) for n in ("nPages", "nRow", "maxPages", "nLayer", "nHead", "headDim", "page",
                                    "block", "kind")]


class GPT2W4(ctypes.Structure):
    """A weight in 4 bits (include/gpt2_b200.h)."""

    _fields_ = [(n, ctypes.c_void_p) for n in ("codes", "scale", "least")] + [(n, ctypes.c_int) for n in ("N", "K", "group")]


class GPT2LogitsEdit(ctypes.Structure):
    """What gpt2_logits_edit_b200 does to each row (include/gpt2_b200.h)."""

    _fields_ = [("repetition", ctypes.c_void_p), ("frequency", ctypes.c_void_p), ("presence", ctypes.c_void_p),
                ("history", ctypes.c_void_p), ("history_stride", ctypes.c_longlong), ("max_history", ctypes.c_int),
                ("length", ctypes.c_void_p), ("prompt", ctypes.c_void_p), ("bias_token", ctypes.c_void_p),
                ("bias", ctypes.c_void_p), ("bias_stride", ctypes.c_longlong), ("max_bias", ctypes.c_int),
                ("n_bias", ctypes.c_void_p), ("mask", ctypes.c_void_p), ("mask_stride", ctypes.c_longlong),
                ("mask_rows", ctypes.c_int), ("mask_row", ctypes.c_void_p)]


class GPT2W4Weights(ctypes.Structure):
    """GPT-2-124M's matmul weights in 4 bits (include/gpt2_b200.h)."""

    _fields_ = [(n, GPT2W4 * N_LAYER) for n in ("qkv", "attn_proj", "fc", "proj")] + [("head", GPT2W4)]


class GPT2LayerGPU(ctypes.Structure):
    """Same layout as GPT2LayerGPU in the reference's cuda/kernels.cuh:19-23."""

    _fields_ = [(n, ctypes.c_void_p) for n, _ in LAYER_TENSORS]


class GPT2WeightsGPU(ctypes.Structure):
    """Same layout as GPT2WeightsGPU in the reference's cuda/kernels.cuh:41-48."""

    _fields_ = [
        ("data", ctypes.c_void_p),
        ("n", ctypes.c_size_t),
        ("wte", ctypes.c_void_p),
        ("wpe", ctypes.c_void_p),
        ("layers", GPT2LayerGPU * N_LAYER),
        ("lnf_g", ctypes.c_void_p),
        ("lnf_b", ctypes.c_void_p),
        ("q", ctypes.c_void_p),
    ]


_vp, _ci, _cll, _cu, _cd = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_uint, ctypes.c_double
_kvp = ctypes.POINTER(GPT2KVCache)
_wp = ctypes.POINTER(GPT2WeightsGPU)
_k8p = ctypes.POINTER(GPT2KV8Cache)
_w4p = ctypes.POINTER(GPT2W4)
_edp = ctypes.POINTER(GPT2LogitsEdit)
_cs = ctypes.c_size_t
_SIGS = {
    "gpt2_attention_b200": (None, [_vp, _vp, _ci, _ci, _ci, _ci]),
    "gpt2_attention_b200_stream": (_ci, [_vp, _vp, _ci, _ci, _ci, _ci, _vp]),
    "gpt2_attention_b200_batched": (_ci, [_vp, _vp, _ci, _ci, _ci, _ci, _ci, _cll, _cll, _vp]),
    "gpt2_attention_kv_b200": (None, [_vp, _vp, _kvp, _ci, _ci, _ci, _ci, _ci]),
    "gpt2_attention_kv_b200_stream": (_ci, [_vp, _vp, _kvp, _ci, _ci, _ci, _ci, _ci, _vp]),
    "gpt2_attn_decode_b200": (None, [_vp, _vp, _kvp, _ci, _ci]),
    "gpt2_attn_decode_b200_stream": (_ci, [_vp, _vp, _kvp, _ci, _ci, _vp]),
    "gpt2_attn_decode_b200_layers": (_ci, [_vp, _cll, _vp, _cll, _kvp, _ci, _ci, _vp, _ci, _ci, _vp]),
    "gpt2_attn_decode_b200_batched": (_ci, [_vp, _cll, _vp, _cll, _vp, _vp, _vp, _ci, _ci, _ci, _ci,
                                            _vp]),
    "gpt2_attn_decode_b200_layers_noalloc": (_ci, [_vp, _cll, _vp, _cll, _kvp, _ci, _ci, _ci, _vp]),
    "gpt2_b200_decode_attn_step": (_ci, [_vp, _cll, _vp, _cll, _kvp, _vp, _ci, _vp]),
    "gpt2_kv_alloc_b200": (_ci, [_kvp, _ci]),
    "gpt2_kv_alloc_shape_b200": (_ci, [_kvp, _ci, _ci, _ci, _ci]),
    "gpt2_kv_free_b200": (None, [_kvp]),
    "gpt2_kv_reset_b200": (None, [_kvp]),
    "gpt2_kv_step_bytes_b200": (_cd, [_kvp, _ci]),
    "gpt2_kv_append_one_b200": (None, [_kvp, _ci, _vp, _ci]),
    "gpt2_kv_append_b200_stream": (_ci, [_kvp, _ci, _ci, _vp, _cll, _vp, _ci, _vp]),
    "gpt2_kv_scatter_prefill_b200": (None, [_kvp, _ci, _vp, _ci]),
    "gpt2_kv_scatter_prefill_b200_stream": (_ci, [_kvp, _ci, _vp, _ci, _vp]),
    "gpt2_decode_step_b200": (None, [_vp, _wp, _kvp, _ci, _ci, _vp, _vp, _vp]),
    "gpt2_b200_batch_create": (_ci, [ctypes.POINTER(_vp), _wp, _kvp, _ci]),
    "gpt2_b200_batch_destroy": (None, [_vp]),
    "gpt2_b200_batch_step": (_ci, [_vp, _vp, _vp, _vp, _cll, _vp, _vp]),
    "gpt2_b200_batch_generate": (_ci, [_vp, _vp, _cll, _vp, _ci, _vp, _cll, _ci, _vp]),
    "gpt2_b200_batch_launches_per_step": (_ci, [_vp, _ci]),
    "gpt2_b200_linear": (_ci, [_vp, _cll, _vp, _cll, _vp, _vp, _ci, _ci, _ci, _ci, _vp]),
    "gpt2_b200_linear_argmax": (_ci, [_vp, _cll, _vp, _cll, _vp, _ci, _ci, _ci, _vp, _vp]),
    "gpt2_gemv_b200": (None, [_vp, _vp, _vp, _vp, _ci, _ci]),
    "gpt2_kv8_work_bytes_b200": (_cs, [_k8p, _ci, _ci]),
    "gpt2_kv8_alloc_b200": (_ci, [_k8p, _ci, _ci]),
    "gpt2_kv8_free_b200": (None, [_k8p]),
    "gpt2_kv8_reset_b200": (_ci, [_k8p, _vp]),
    "gpt2_kv8_store_b200": (_ci, [_k8p, _ci, _ci, _vp, _vp, _cll, _cll, _cll, _vp, _ci, _vp]),
    "gpt2_kv8_load_b200": (_ci, [_k8p, _ci, _ci, _vp, _vp, _cll, _cll, _cll, _vp, _ci, _vp, _ci, _vp]),
    "gpt2_kv8_attend_b200": (_ci, [_vp, _cll, _cll, _vp, _cll, _cll, _k8p, _ci, _ci, _ci, _vp, _vp, _ci,
                                   _ci, _vp]),
    "gpt2_kv8_reorder_b200": (_ci, [_k8p, _vp, _ci, _ci, _vp]),
    "gpt2_kv8_compact_b200": (_ci, [_k8p, _vp, _vp]),
    "gpt2_beam_work_bytes_b200": (_cs, [_ci, _ci]),
    "gpt2_beam_select_b200": (_ci, [_vp, _vp, _vp, _vp, _vp, _ci, _cll, _vp, _vp, _ci, _ci, _ci, _ci, _vp,
                                    _cs, _vp]),
    "gpt2_b200_beam_create": (_ci, [ctypes.POINTER(_vp), _wp, _k8p, _ci, _ci]),
    "gpt2_b200_beam_destroy": (None, [_vp]),
    "gpt2_b200_beam_generate": (_ci, [_vp, _vp, _cll, _vp, _ci, _ci, _vp, _cll, _vp, _vp]),
    "gpt2_w4_quantize_b200": (_ci, [_w4p, _vp, _cll, _vp]),
    "gpt2_w4_dequantize_b200": (_ci, [_vp, _cll, _w4p, _vp]),
    "gpt2_w4_linear_b200": (_ci, [_vp, _cll, _vp, _cll, _w4p, _vp, _vp, _cll, _ci, _ci, _vp]),
    "gpt2_logits_edit_b200": (_ci, [_vp, _cll, _vp, _cll, _ci, _ci, _ci, _edp, _vp, _vp]),
    "gpt2_b200_batch_create_w4": (_ci, [ctypes.POINTER(_vp), _wp, ctypes.POINTER(GPT2W4Weights), _kvp, _ci]),
    "gpt2_b200_batch_generate_edited": (_ci, [_vp, _vp, _cll, _vp, _ci, _vp, _cll, _edp, _vp]),
    "gpt2_b200_compose_backend": (None, [ctypes.POINTER(GPT2Backend), ctypes.POINTER(GPT2Backend)]),
    "gpt2_b200_reserve": (_ci, [_ci, _ci, _ci]),
    "gpt2_b200_status": (_cu, [_ci]),
    "gpt2_b200_last_error": (_ci, []),
    "gpt2_b200_strerror": (ctypes.c_char_p, [_ci]),
    "gpt2_b200_selftest_wait_timeout": (_ci, [_cu]),
    "gpt2_b200_version": (ctypes.c_char_p, []),
}


def header_functions(path: str = HEADER) -> list[str]:
    """Names of every function the C header declares (for the export check)."""
    text = open(path).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    names = re.findall(r"^[A-Za-z_][\w \*]*?\b(gpt2_\w+)\s*\(", text, flags=re.M)
    return sorted(set(names))


class Lib:
    """The loaded library with typed entry points (attribute access = C function)."""

    def __init__(self, path: str = LIB_PATH):
        if not os.path.exists(path):
            raise FileNotFoundError(
                f"{path} is missing: build it with `make -C bare-metal-gpt2_b200` (there is no "
                "fallback implementation)")
        self.path = path
        self.lib = ctypes.CDLL(path)
        for name, (res, args) in _SIGS.items():
            fn = getattr(self.lib, name)
            fn.restype = res
            fn.argtypes = args
        self._beam_select = self.lib.gpt2_beam_select_b200

    def __getattr__(self, name):
        return getattr(self.lib, name)

    # -------------------------------------------------------------- checked helpers
    def check(self, rc: int, what: str) -> None:
        """Raises RuntimeError with the library's message for any return code other than OK."""
        if rc != OK:
            raise RuntimeError(f"{what}: {self.lib.gpt2_b200_strerror(rc).decode()} ({rc})")

    def prefill(self, att, qkv, T: int, B: int = 1, stream: int = 0, qkv_stride: int = 0,
                att_stride: int = 0, E: int = 768, H: int = 12) -> None:
        """Causal prefill attention of B sequences (or layers) of T rows: att[b] from qkv[b] as the
        reference's attention slot computes it (cuda/kernels_fused.cu:145-149, one launch for all B).
        Strides are in elements, 0 for packed rows."""
        rc = self.lib.gpt2_attention_b200_batched(att.data_ptr(), qkv.data_ptr(), B, T, E, H, 64,
                                                  qkv_stride, att_stride, stream)
        self.check(rc, "gpt2_attention_b200_batched")

    def decode_layers(self, att, att_stride: int, q, q_stride: int, kv: GPT2KVCache, L0: int,
                      nL: int, length: int = 0, d_len=None, max_len: int = 0,
                      stream: int = 0) -> None:
        """M=1 decode attention of layers L0..L0+nL-1 over the first `length` cache positions (or the
        device int `d_len`), one launch: gpt2_attn_decode (cuda/kvcache.cu:207-210) for many layers."""
        rc = self.lib.gpt2_attn_decode_b200_layers(
            att.data_ptr(), att_stride, q.data_ptr(), q_stride, ctypes.byref(kv), L0, nL,
            d_len.data_ptr() if d_len is not None else None, length, max_len, stream)
        self.check(rc, "gpt2_attn_decode_b200_layers")

    def beam_work(self, torch, B: int, W: int, device):
        """The zeroed scratch of beam_select for B items of W beams."""
        return torch.zeros(self.lib.gpt2_beam_work_bytes_b200(B, W), dtype=torch.uint8, device=device)

    def beam_select(self, token, parent, new_score, new_done, logits, score, done, B: int, W: int,
                    eos: int, work, stream: int = 0) -> None:
        """The W best continuations of each of B items' W beams: logits [B*W][V] fp16 or fp32 (rows may be
        strided), score fp32 [B*W], done int32 [B*W] or None; writes token and parent (int32), new_score
        and new_done (may be score and done; new_done may be None)."""
        i32, f32, kinds, u8 = _types()
        kind, strides, shape, n = kinds.get(logits.dtype), logits.stride(), logits.shape, B * W
        if kind is None or len(strides) != 2 or strides[1] != 1 or shape[0] != n:
            raise ValueError("beam_select: logits are fp16 or fp32, B * W rows of neighbouring values")
        at, what = logits.device, "beam_select"
        rc = self._beam_select(
            _vector(what, token, i32, n, at), _vector(what, parent, i32, n, at), _vector(what, new_score, f32, n, at),
            _vector(what, new_done, i32, n, at) if new_done is not None else None, logits.data_ptr(), kind, strides[0],
            _vector(what, score, f32, n, at), _vector(what, done, i32, n, at) if done is not None else None,
            B, W, shape[1], eos, _vector(what, work, u8, work.numel(), at), work.numel(), stream)
        if rc:
            self.check(rc, "gpt2_beam_select_b200")

    def status(self, clear: bool = True) -> int:
        """The device's status word (bounded-wait timeouts and bad-input bits), cleared if asked."""
        return int(self.lib.gpt2_b200_status(1 if clear else 0))


def cache_view(data_ptr: int, n_layer: int, max_t: int, n_head: int = 12, head_dim: int = 64,
               length: int = 0) -> GPT2KVCache:
    """A GPT2KVCache describing an existing device arena (e.g. a torch tensor's storage)."""
    kv = GPT2KVCache()
    kv.data = data_ptr
    kv.maxT = max_t
    kv.nLayer = n_layer
    kv.nHead = n_head
    kv.headDim = head_dim
    kv.bytes = 2 * n_layer * n_head * max_t * head_dim * 2
    kv.len = length
    return kv


class KV8Cache:
    """A paged 8-bit KV cache over torch tensors (GPT2KV8Cache and the gpt2_kv8_* entry points).

    data uint8 [pages][layers][2][heads][page][dim], scale fp32 [pages][layers][2][heads][page/block], ref
    int32 [pages], table int32 [rows][max pages], length int32 [rows]; the tensors stay alive with the
    cache. q_heads and queries bound what attend() may be called with. create() makes an empty one.
    """

    def __init__(self, lib: "Lib", torch, data, scale, ref, table, length, kind: str = "int8",
                 q_heads: int = 0, queries: int = 1):
        self.lib, self.kind = lib, kind
        n_pages, n_layer, two, n_head, page, dim = data.shape
        shapes = (tuple(scale.shape[:4]) == (n_pages, n_layer, 2, n_head) and two == 2
                  and page % max(1, scale.shape[4]) == 0 and tuple(ref.shape) == (n_pages,)
                  and tuple(length.shape) == (table.shape[0],))
        types = (data.dtype == torch.uint8 and scale.dtype == torch.float32
                 and ref.dtype == table.dtype == length.dtype == torch.int32)
        if not shapes or not types or not all(t.is_contiguous() and t.device == data.device
                                              for t in (data, scale, ref, table, length)):
            raise ValueError("KV8Cache: data, scale, ref, table or length has another shape, type, layout or device")
        self.data, self.scale, self.ref, self.table, self.length = data, scale, ref, table, length
        c = GPT2KV8Cache()
        c.data, c.scale, c.ref = data.data_ptr(), scale.data_ptr(), ref.data_ptr()
        c.table, c.len = table.data_ptr(), length.data_ptr()
        c.nPages, c.nLayer, c.nHead, c.headDim, c.page = n_pages, n_layer, n_head, dim, page
        c.nRow, c.maxPages = table.shape
        c.block, c.kind = page // max(1, scale.shape[4]), KV8_KINDS[kind]
        n = lib.gpt2_kv8_work_bytes_b200(ctypes.byref(c), q_heads or n_head, queries)
        if not n:
            raise ValueError("KV8Cache: a shape outside the supported ones")
        self.work = torch.zeros(n, dtype=torch.uint8, device=data.device)
        c.work, c.work_bytes = self.work.data_ptr(), n
        self.c, self.ref_c = c, ctypes.byref(c)
        # what every call needs, looked up once: a decoding step makes dozens of calls
        self._nrow, self._dim, self._width, self._half = int(c.nRow), dim, n_head * dim, torch.float16
        self._at, self._int = data.device, torch.int32
        self._store, self._load = lib.lib.gpt2_kv8_store_b200, lib.lib.gpt2_kv8_load_b200
        self._attend, self._reorder = lib.lib.gpt2_kv8_attend_b200, lib.lib.gpt2_kv8_reorder_b200
        self._compact = lib.lib.gpt2_kv8_compact_b200

    @classmethod
    def create(cls, lib: "Lib", torch, rows: int, max_pages: int, pages: int, layers: int = N_LAYER,
               heads: int = N_HEAD, dim: int = 64, page: int = 16, block: int = 16, kind: str = "int8",
               q_heads: int = 0, queries: int = 1, device="cuda") -> "KV8Cache":
        """An empty cache: every page free, every row without positions."""
        z = dict(device=device, dtype=torch.int32)
        return cls(lib, torch, torch.zeros(pages, layers, 2, heads, page, dim, device=device, dtype=torch.uint8),
                   torch.zeros(pages, layers, 2, heads, page // block, device=device),
                   torch.zeros(pages, **z), torch.full((rows, max_pages), -1, **z), torch.zeros(rows, **z),
                   kind, q_heads, queries)

    def _rows(self, what, k, v):
        """The three outer strides of k and v and their tokens, after a check of their form."""
        s, shape = k.stride(), k.shape
        if s != v.stride() or shape != v.shape or len(s) != 4 or s[3] != 1 or shape[1] != self._nrow or \
                shape[3] != self._width or k.dtype != self._half or v.dtype != self._half or \
                k.device != self._at or v.device != self._at:
            raise ValueError(f"{what}: k and v are fp16 [layers][rows][tokens][heads * dim], laid out alike, on the "
                             "cache's device")
        return shape[0], s[0], s[1], s[2], shape[2]

    def _per_row(self, what, t):
        return _vector(what, t, self._int, self._nrow, self._at)

    def _count(self, what, count):
        """(int, device pointer or None) of a count given as an int, an int32 tensor or None."""
        if count is None:
            return 0, None
        return (count, None) if isinstance(count, int) else (0, self._per_row(what, count))

    def store(self, k, v, layer: int = 0, count=None, stream: int = 0) -> None:
        """k, v: fp16 [layers][rows][tokens][heads * dim] (strided views are fine), written behind the
        held positions from `layer` on; count: int32 [rows] or None (all tokens)."""
        n, ls, rs, ts, tokens = self._rows("store", k, v)
        rc = self._store(self.ref_c, layer, n, k.data_ptr(), v.data_ptr(), ls, rs, ts,
                         self._per_row("store", count) if count is not None else None, tokens, stream)
        if rc:
            self.lib.check(rc, "gpt2_kv8_store_b200")

    def load(self, k, v, layer: int = 0, first=None, count=None, stream: int = 0) -> None:
        """The inverse: positions first[r].. (0 without first) as fp16 rows, 0 beyond the held ones;
        count: int32 [rows], an int or None: positions stored but not yet counted in."""
        n, ls, rs, ts, tokens = self._rows("load", k, v)
        add, d_add = self._count("load", count)
        rc = self._load(self.ref_c, layer, n, k.data_ptr(), v.data_ptr(), ls, rs, ts,
                        self._per_row("load", first) if first is not None else None, tokens, d_add, add, stream)
        if rc:
            self.lib.check(rc, "gpt2_kv8_load_b200")

    def attend(self, out, q, layer: int = 0, count=None, first=None, max_len: int = 0,
               stream: int = 0) -> None:
        """q, out: fp16 [rows][queries][q heads * dim]: causal attention of each row's last positions over
        its keys, counted as load() counts them; keys before first[r] are masked."""
        qs, os_, shape = q.stride(), out.stride(), q.shape
        if shape != out.shape or len(qs) != 3 or shape[0] != self._nrow or qs[2] != 1 or os_[2] != 1 or \
                shape[2] % self._dim or q.dtype != self._half or out.dtype != self._half or \
                q.device != self._at or out.device != self._at:
            raise ValueError("attend: q and out are fp16 [rows][queries][q heads * dim] on the cache's device")
        add, d_add = self._count("attend", count)
        rc = self._attend(out.data_ptr(), os_[0], os_[1], q.data_ptr(), qs[0], qs[1], self.ref_c, layer,
                          shape[2] // self._dim, shape[1],
                          self._per_row("attend", first) if first is not None else None, d_add, add, max_len, stream)
        if rc:
            self.lib.check(rc, "gpt2_kv8_attend_b200")

    def reorder(self, parent=None, advance: int = 0, reserve: int = 0, stream: int = 0) -> None:
        """Counts `advance` positions in, makes row r a copy of row parent[r] (int32 [rows]; -1: empty; None:
        itself) by sharing pages, and makes room for `reserve` more positions."""
        rc = self._reorder(self.ref_c, self._per_row("reorder", parent) if parent is not None else None, advance,
                           reserve, stream)
        if rc:
            self.lib.check(rc, "gpt2_kv8_reorder_b200")

    def compact(self, live=None, stream: int = 0) -> None:
        """Moves the live pages to the lowest ids; live: int32 [1] for their number, or None."""
        rc = self._compact(self.ref_c, _vector("compact", live, self._int, 1, self._at) if live is not None else None,
                           stream)
        if rc:
            self.lib.check(rc, "gpt2_kv8_compact_b200")

    def reset(self, stream: int = 0) -> None:
        """Every page free, every row empty."""
        self.lib.check(self.lib.gpt2_kv8_reset_b200(self.ref_c, stream), "gpt2_kv8_reset_b200")


class W4Weight:
    """A weight [N][K] in 4 bits over torch tensors (GPT2W4 and the gpt2_w4_* entry points).

    codes uint8 [N][K/2], scale fp16 [K/group][N], least fp16 [K/group][N] or None; the tensors stay alive with the
    weight. create() makes an empty one, pack() one from an fp16 weight.
    """

    def __init__(self, lib: "Lib", torch, codes, scale, least=None):
        tensors = [t for t in (codes, scale, least) if t is not None]
        if codes.dim() != 2 or scale.dim() != 2 or (least is not None and least.shape != scale.shape) or codes.dtype != torch.uint8 or \
                any(t.dtype != torch.float16 for t in tensors[1:]) or not all(t.is_contiguous() and t.device == codes.device for t in tensors):
            raise ValueError("W4Weight: codes are uint8 [N][K/2], scale and least fp16 [K/group][N], contiguous on one device")
        N, K = codes.shape[0], 2 * codes.shape[1]
        group = K // max(1, scale.shape[0])
        if group not in (32, 64, 128) or K % group or scale.shape != (K // group, N) or N < 1:
            raise ValueError("W4Weight: groups of 32, 64 or 128 neighbouring k, one scale per group and row")
        self.lib, self.N, self.K, self.group = lib, N, K, group
        self.codes, self.scale, self.least = codes, scale, least
        c = GPT2W4()
        c.codes, c.scale, c.least = codes.data_ptr(), scale.data_ptr(), least.data_ptr() if least is not None else None
        c.N, c.K, c.group = N, K, group
        self.c, self.ref_c = c, ctypes.byref(c)
        self._at, self._half, self._current = codes.device, torch.float16, _current(torch, codes.device)
        self._quantize, self._dequantize, self._linear = (_entry(call, codes.device) for call in (
            lib.lib.gpt2_w4_quantize_b200, lib.lib.gpt2_w4_dequantize_b200, lib.lib.gpt2_w4_linear_b200))

    @classmethod
    def create(cls, lib: "Lib", torch, N: int, K: int, group: int = 64, least: bool = False, device="cuda") -> "W4Weight":
        """An empty weight; least: the form with a smallest value per group."""
        if group not in (32, 64, 128) or K < 1 or K % group:
            raise ValueError("W4Weight: K is a multiple of the group, which is 32, 64 or 128")
        at = dict(device=device, dtype=torch.float16)
        return cls(lib, torch, torch.zeros(N, K // 2, device=device, dtype=torch.uint8), torch.zeros(K // group, N, **at),
                   torch.zeros(K // group, N, **at) if least else None)

    @classmethod
    def pack(cls, lib: "Lib", torch, w, group: int = 64, least: bool = False, stream: int = 0) -> "W4Weight":
        """The fp16 weight w [N][K] in 4 bits. `stream` first waits for torch's current stream, on which w was made and the weight's
        memory comes from the allocator."""
        q = cls.create(lib, torch, w.shape[0], w.shape[1], group, least, w.device)
        if w.device.type == "cuda":
            current = torch.cuda.current_stream(w.device)
            if stream != current.cuda_stream:
                st = torch.cuda.ExternalStream(stream, w.device) if stream else torch.cuda.default_stream(w.device)
                st.wait_stream(current)
                for t in (w, q.codes, q.scale, q.least):
                    if t is not None:
                        t.record_stream(st)
        q.quantize(w, stream)
        return q

    def _matrix(self, what, w):
        if w.dtype != self._half or w.dim() != 2 or w.shape != (self.N, self.K) or w.stride(1) != 1 or w.device != self._at:
            raise ValueError(f"{what}: expected fp16 [{self.N}][{self.K}] on the weight's device")
        self._current(what)
        return w.data_ptr(), w.stride(0) if self.N > 1 else self.K

    def quantize(self, w, stream: int = 0) -> None:
        """Writes the codes, scales and least values of the fp16 weight w [N][K]."""
        p, ld = self._matrix("quantize", w)
        self.lib.check(self._quantize(self.ref_c, p, ld, stream), "gpt2_w4_quantize_b200")

    def dequantize(self, w, stream: int = 0) -> None:
        """Writes the fp16 values that the codes stand for to w [N][K]."""
        p, ld = self._matrix("dequantize", w)
        self.lib.check(self._dequantize(p, ld, self.ref_c, stream), "gpt2_w4_dequantize_b200")

    def linear(self, out, x, bias=None, epi: int = LINEAR_STORE, residual=None, stream: int = 0) -> None:
        """out [B][N] = e(x [B][K] W^T + bias [N]), fp16 rows (strided ones are fine); epi LINEAR_RESID adds residual [B][N]
        (None: what out holds)."""
        shape, os_, xs, half, at = out.shape, out.stride(), x.stride(), self._half, self._at
        B = shape[0] if len(shape) == 2 else 0
        if B < 1 or shape[1] != self.N or x.shape != (B, self.K) or xs[1] != 1 or (os_[1] != 1 and self.N > 1) or x.dtype is not half or \
                out.dtype is not half or x.device != at or out.device != at:
            raise ValueError("linear: out is fp16 [B][N] and x fp16 [B][K] on the weight's device")
        rp, rs = None, 0
        if epi == LINEAR_RESID:
            r = out if residual is None else residual
            rs = r.stride()
            if r.shape != shape or (rs[1] != 1 and self.N > 1) or r.dtype is not half or r.device != at:
                raise ValueError("linear: residual is fp16 [B][N] on the weight's device")
            rp, rs = r.data_ptr(), rs[0] if B > 1 else self.N
        self._current("linear")
        rc = self._linear(out.data_ptr(), os_[0] if B > 1 else self.N, x.data_ptr(), xs[0] if B > 1 else self.K, self.ref_c,
                          _vector("linear", bias, half, self.N, at) if bias is not None else None, rp, rs, B, epi, stream)
        if rc:
            self.lib.check(rc, "gpt2_w4_linear_b200")


class LogitsEdit:
    """Penalties, biases and masks of a batch of rows (GPT2LogitsEdit and gpt2_logits_edit_b200), over tensors that the
    program fills and changes between calls; they stay alive with the edit.

    repetition, frequency, presence fp32 [rows] or None; history int32 [rows][most] (its first length[r] tokens count, all without
    length; the first prompt[r] of them are the prompt); bias_token int32 and bias fp32 [rows][most] (n_bias int32 [rows] of them, or
    all); mask int32 [mask rows][>= ceil(vocab / 32)], bit t % 32 of word t / 32 set where t is allowed; mask_row int32
    [rows] names each row's (-1: none), by default its own, or the only one.
    """

    def __init__(self, lib: "Lib", torch, rows: int, vocab: int, repetition=None, frequency=None, presence=None, history=None, length=None,
                 prompt=None, bias_token=None, bias=None, n_bias=None, mask=None, mask_row=None):
        tensors = (repetition, frequency, presence, history, length, prompt, bias_token, bias, n_bias, mask, mask_row)
        some = [t for t in tensors if t is not None]
        self.lib, self.rows, self.vocab, self.tensors = lib, rows, vocab, tensors
        self._at = self.device = some[0].device if some else None
        i32, f32, self._kinds, _ = _types()
        e = GPT2LogitsEdit()
        for name, t, kind in (("repetition", repetition, f32), ("frequency", frequency, f32), ("presence", presence, f32), ("length", length, i32),
                              ("prompt", prompt, i32), ("n_bias", n_bias, i32), ("mask_row", mask_row, i32)):
            if t is not None:
                setattr(e, name, _vector("LogitsEdit", t, kind, rows, self._at))

        def table(name, t, kind, n):
            if t.dim() != 2 or t.dtype is not kind or t.shape[0] != n or t.device != self._at or (t.shape[1] > 1 and t.stride(1) != 1):
                raise ValueError(f"LogitsEdit: {name} is {kind} with {n} rows of neighbouring values on the others' device")
            stride = t.stride(0) if n > 1 else t.shape[1]
            if 0 < stride < t.shape[1]:
                raise ValueError(f"LogitsEdit: the rows of {name} overlap")
            return t.data_ptr(), stride, t.shape[1]

        if history is not None:
            e.history, e.history_stride, e.max_history = table("history", history, i32, rows)
        elif length is not None or prompt is not None:
            raise ValueError("LogitsEdit: length and prompt belong to a history")
        if (bias is None) != (bias_token is None) or (bias is None and n_bias is not None):
            raise ValueError("LogitsEdit: bias_token, bias and n_bias belong together")
        if bias is not None:
            if bias.shape != bias_token.shape or bias.stride() != bias_token.stride():
                raise ValueError("LogitsEdit: bias_token and bias are laid out alike")
            e.bias_token, e.bias_stride, e.max_bias = table("bias_token", bias_token, i32, rows)
            e.bias = table("bias", bias, f32, rows)[0]
        if mask is not None:
            n = mask.shape[0]
            e.mask, stride, words = table("mask", mask, i32, n)
            if n > 1 and stride == 0:  # the same for all rows
                if mask_row is not None or n != rows:
                    raise ValueError("LogitsEdit: mask_row names rows of their own")
                n = 1
            if words < (vocab + 31) // 32 or (mask_row is None and n not in (1, rows)):
                raise ValueError("LogitsEdit: a mask has a bit for each token, and one row, as many as the edit, or mask_row")
            e.mask_rows, e.mask_stride = n, stride or words
        elif mask_row is not None:
            raise ValueError("LogitsEdit: mask_row belongs to a mask")
        self.c, self.ref_c = e, ctypes.byref(e)
        self._torch, self._current = torch, _current(torch, self._at) if some else None
        self._edit = _entry(lib.lib.gpt2_logits_edit_b200, self._at)

    def apply(self, out, logits, next_tokens=None, stream: int = 0) -> None:
        """out [rows][vocab] = the edited logits (fp16 or fp32 rows, strided ones are fine; out may be logits); next_tokens int32
        [rows]: each row's largest, or None."""
        kind, shape, os_, ls, at = self._kinds.get(logits.dtype), logits.shape, out.stride(), logits.stride(), logits.device
        rows, vocab = self.rows, self.vocab
        if kind is None or out.dtype is not logits.dtype or len(shape) != 2 or shape[0] != rows or shape[1] != vocab or out.shape != shape or \
                (vocab > 1 and (ls[1] != 1 or os_[1] != 1)) or out.device != at or (self._at is not None and at != self._at):
            raise ValueError("apply: logits and out are fp16 or fp32 [rows][vocab] of one type, on the edit's device")
        if self._current is not None:
            self._current("apply")
        else:  # no tensors of its own: the logits say where
            _on_gpu("apply", at)
            _current(self._torch, at)("apply")
        rc = self._edit(out.data_ptr(), os_[0] if rows > 1 else vocab, logits.data_ptr(), ls[0] if rows > 1 else vocab, kind, rows, vocab, self.ref_c,
                        _vector("apply", next_tokens, _types()[0], rows, at) if next_tokens is not None else None, stream)
        if rc:
            self.lib.check(rc, "gpt2_logits_edit_b200")


class ModelWeights:
    """Seeded random GPT-2-124M fp16 weights in one device buffer, described by a GPT2WeightsGPU.

    hf_init=True follows GPT-2's initialisation (linear weights and embeddings N(0, std), biases 0,
    LayerNorm gain 1 and bias 0); hf_init=False also randomises the biases and LayerNorm parameters
    so that every epilogue term is exercised (tests).
    """

    def __init__(self, torch, device, seed: int = 0, std: float = 0.02, hf_init: bool = True):
        shapes = [("wte", (VOCAB, N_EMBD)), ("wpe", (N_CTX, N_EMBD))]
        shapes += [(f"h{L}.{n}", sh) for L in range(N_LAYER) for n, sh in LAYER_TENSORS]
        shapes += [("lnf_g", (N_EMBD,)), ("lnf_b", (N_EMBD,))]
        total = sum(_numel(sh) for _, sh in shapes)
        self.buf = torch.empty(total, dtype=torch.float16, device=device)
        gen = torch.Generator(device=device)
        gen.manual_seed(seed)
        self.t = {}
        off = 0
        for name, sh in shapes:
            n = _numel(sh)
            v = self.buf[off:off + n].view(sh)
            off += n
            if name.endswith("_g"):
                v.fill_(1.0)
                if not hf_init:
                    v.add_(0.1 * torch.randn(sh, generator=gen, device=device))
            elif name.endswith("_b"):
                if hf_init:
                    v.zero_()
                else:
                    v.copy_(std * torch.randn(sh, generator=gen, device=device))
            else:
                v.copy_(std * torch.randn(sh, generator=gen, device=device))
            self.t[name] = v
        w = GPT2WeightsGPU()
        w.data = self.buf.data_ptr()
        w.n = total
        w.wte = self.t["wte"].data_ptr()
        w.wpe = self.t["wpe"].data_ptr()
        for L in range(N_LAYER):
            for n, _ in LAYER_TENSORS:
                setattr(w.layers[L], n, self.t[f"h{L}.{n}"].data_ptr())
        w.lnf_g = self.t["lnf_g"].data_ptr()
        w.lnf_b = self.t["lnf_b"].data_ptr()
        w.q = None
        self.struct = w


class W4ModelWeights:
    """The matmul weights of a ModelWeights in 4 bits (GPT2W4Weights): `layers` holds a W4Weight per layer and name, `head` the tied
    head's, or None with head=False (the fp16 embedding is the head then)."""

    NAMES = (("qkv", "qkv_w"), ("attn_proj", "attn_proj_w"), ("fc", "fc_w"), ("proj", "proj_w"))

    def __init__(self, lib: "Lib", torch, weights: ModelWeights, group: int = 64, least: bool = False, head: bool = True, stream: int = 0):
        self.struct = GPT2W4Weights()
        self.layers = []
        for L in range(N_LAYER):
            q = {n: W4Weight.pack(lib, torch, weights.t[f"h{L}.{t}"], group, least, stream) for n, t in self.NAMES}
            for n, _ in self.NAMES:
                getattr(self.struct, n)[L] = q[n].c
            self.layers.append(q)
        self.head = W4Weight.pack(lib, torch, weights.t["wte"], group, least, stream) if head else None
        if head:
            self.struct.head = self.head.c


class DecodeBatch:
    """B sequences of GPT-2-124M decoded together (the gpt2_b200_batch_* entry points).

    caches: a torch fp16 tensor [B][12][2][12][maxT][64] (each sequence's arena in the reference
    layout) that stays alive as long as the batch. step() consumes one token per sequence at its
    position; generate() runs lock-step greedy generation (prompt tokens first) in a CUDA graph.
    w4: the matmuls run over these 4-bit weights instead of the weights' own.
    """

    def __init__(self, lib: "Lib", weights: ModelWeights, caches, w4: "W4ModelWeights | None" = None):
        if w4 is not None and any(q.codes.device != caches.device for q in [*(q for layer in w4.layers for q in layer.values()), w4.head] if q is not None):
            raise ValueError(f"DecodeBatch: the 4-bit weights are on another device than the caches, {caches.device}")
        self.lib, self.weights, self.caches, self.w4 = lib, weights, caches, w4
        self.B, max_t = int(caches.shape[0]), int(caches.shape[4])
        self.kvs = (GPT2KVCache * self.B)(*[cache_view(caches[b].data_ptr(), N_LAYER, max_t)
                                             for b in range(self.B)])
        self.h = ctypes.c_void_p()
        if w4 is not None:
            lib.check(lib.gpt2_b200_batch_create_w4(ctypes.byref(self.h), ctypes.byref(weights.struct), ctypes.byref(w4.struct),
                                                    self.kvs, self.B), "gpt2_b200_batch_create_w4")
            return
        lib.check(lib.gpt2_b200_batch_create(ctypes.byref(self.h), ctypes.byref(weights.struct),
                                             self.kvs, self.B), "gpt2_b200_batch_create")

    def step(self, tokens, positions, logits=None, next_tokens=None, stream: int = 0) -> None:
        """tokens, positions: int32 device tensors [B]; logits: fp16 [B][>= VOCAB] or None;
        next_tokens: int32 [B] or None (argmax of each row)."""
        self.lib.check(self.lib.gpt2_b200_batch_step(
            self.h, tokens.data_ptr(), positions.data_ptr(),
            logits.data_ptr() if logits is not None else None,
            logits.stride(0) if logits is not None else 0,
            next_tokens.data_ptr() if next_tokens is not None else None, stream),
            "gpt2_b200_batch_step")

    def generate(self, prompt, prompt_len, n_steps: int, out, stream: int = 0, edit: "LogitsEdit | None" = None) -> None:
        """prompt: int32 [B][P]; prompt_len: int32 [B] (1..P); out: int32 [B][>= n_steps+1]. edit: made for B rows of VOCAB
        logits without a history; every choice is made of the logits so edited, out and prompt_len being the history. All steps are enqueued
        here: what the edit's tensors hold is the same for all of them."""
        if edit is not None:
            if edit.rows != self.B or edit.vocab != VOCAB or edit.c.history:
                raise ValueError("generate: edit is for the batch's rows of VOCAB logits, without a history of its own")
            i32, at = _types()[0], self.caches.device
            for t in (prompt, out):
                if t.dim() != 2 or t.dtype is not i32 or t.shape[0] != self.B or t.shape[1] < 1 or t.stride(1) != 1 or t.device != at:
                    raise ValueError("generate: prompt is int32 [B][P], out int32 [B][>= n_steps + 1], on the caches' device")
            if out.shape[1] <= n_steps or (edit.device is not None and edit.device != at):
                raise ValueError("generate: out is too narrow, or the edit is on another device")
            self.edit = edit  # its tensors are read by steps that run behind this call
            self.lib.check(self.lib.gpt2_b200_batch_generate_edited(
                self.h, prompt.data_ptr(), _row_stride(prompt), _vector("generate", prompt_len, i32, self.B, at), n_steps, out.data_ptr(),
                _row_stride(out), edit.ref_c, stream), "gpt2_b200_batch_generate_edited")
            return
        self.lib.check(self.lib.gpt2_b200_batch_generate(
            self.h, prompt.data_ptr(), _row_stride(prompt), prompt_len.data_ptr(), n_steps,
            out.data_ptr(), _row_stride(out), 0, stream), "gpt2_b200_batch_generate")

    def close(self) -> None:
        """Destroys the batch (the library synchronises the device first); safe to call twice."""
        if self.h:
            self.lib.gpt2_b200_batch_destroy(self.h)
            self.h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:  # noqa: BLE001 - interpreter shutdown
            pass


class BeamDecoder:
    """Beam search with GPT-2-124M over a KV8Cache of B * W rows (the gpt2_b200_beam_* entry points)."""

    def __init__(self, lib: "Lib", weights: ModelWeights, cache: KV8Cache, B: int, W: int):
        self.lib, self.weights, self.cache, self.B, self.W = lib, weights, cache, B, W
        self.h = ctypes.c_void_p()
        lib.check(lib.gpt2_b200_beam_create(ctypes.byref(self.h), ctypes.byref(weights.struct), cache.ref_c, B, W),
                  "gpt2_b200_beam_create")

    def generate(self, prompt, prompt_len, n_steps: int, out, score=None, eos: int = -1, stream: int = 0) -> None:
        """prompt: int32 [B][P]; prompt_len: int32 [B] (1..P); out: int32 [B * W][>= n_steps+1], each item's
        hypotheses best first; score: fp32 [B * W] or None."""
        i32, f32, _, _ = _types()
        at, rows, what = self.cache.data.device, self.B * self.W, "generate"
        for t, n in ((prompt, self.B), (out, rows)):
            if t.dim() != 2 or t.dtype is not i32 or t.shape[0] != n or t.shape[1] < 1 or t.stride(1) != 1 or t.device != at:
                raise ValueError("generate: prompt is int32 [B][P], out int32 [B * W][>= n_steps + 1], on the cache's device")
        if out.shape[1] <= n_steps < _row_stride(out):  # a view whose rows end early: the library sees the stride alone
            raise ValueError("generate: out is too narrow")
        self.lib.check(self.lib.gpt2_b200_beam_generate(
            self.h, prompt.data_ptr(), _row_stride(prompt), _vector(what, prompt_len, i32, self.B, at), n_steps, eos, out.data_ptr(),
            _row_stride(out), _vector(what, score, f32, rows, at) if score is not None else None, stream), "gpt2_b200_beam_generate")

    def close(self) -> None:
        """Destroys the decoder (the library synchronises the device first); safe to call twice."""
        if self.h:
            self.lib.gpt2_b200_beam_destroy(self.h)
            self.h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:  # noqa: BLE001 - interpreter shutdown
            pass


def _current(torch, device):
    """A check that the calling thread's current device is `device`: the library launches there."""
    get, index = torch.cuda.current_device, device.index
    if device.type != "cuda":
        return lambda what: None

    def check(what):
        if get() != index:
            raise ValueError(f"{what}: the tensors are on {device}, the current device is cuda:{get()}")
    return check


def _on_gpu(what, device) -> None:
    if device.type != "cuda":
        raise ValueError(f"{what}: the tensors are on {device}, the library takes those of a GPU")


def _entry(call, device):
    """The library's call; where the tensors are not on a GPU, one that refuses their addresses. device None: not known yet."""
    if device is None or device.type == "cuda":
        return call
    return lambda *a: _on_gpu(call.__name__, device)


def _row_stride(t) -> int:
    """The elements from a matrix's row to the next; of a single row, whose stride may be anything, its width at least."""
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[-1])


def _vector(what, t, dtype, n, device):
    """The address of t, which must hold n neighbouring elements of the type on the device."""
    if t.dtype is not dtype or t.numel() != n or t.device != device or not t.is_contiguous():
        raise ValueError(f"{what}: expected {n} neighbouring {dtype} on the device of the other tensors, got "
                         f"{tuple(t.shape)} {t.dtype} on {t.device}")
    return t.data_ptr()


_TYPES: list = []


def _types():
    """torch.int32, torch.float32, and the types of logits."""
    if not _TYPES:
        import torch
        _TYPES.extend((torch.int32, torch.float32, {torch.float16: BEAM_HALF, torch.float32: BEAM_FLOAT}, torch.uint8))
    return _TYPES


def _numel(shape) -> int:
    n = 1
    for d in shape:
        n *= d
    return n


_LIB: Lib | None = None


def load() -> Lib:
    """The process-wide Lib; raises if lib/libgpt2_b200.so is missing (there is no fallback)."""
    global _LIB
    if _LIB is None:
        _LIB = Lib()
    return _LIB
