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


class DecodeBatch:
    """B sequences of GPT-2-124M decoded together (the gpt2_b200_batch_* entry points).

    caches: a torch fp16 tensor [B][12][2][12][maxT][64] (each sequence's arena in the reference
    layout) that stays alive as long as the batch. step() consumes one token per sequence at its
    position; generate() runs lock-step greedy generation (prompt tokens first) in a CUDA graph.
    """

    def __init__(self, lib: "Lib", weights: ModelWeights, caches):
        self.lib, self.weights, self.caches = lib, weights, caches
        self.B, max_t = int(caches.shape[0]), int(caches.shape[4])
        self.kvs = (GPT2KVCache * self.B)(*[cache_view(caches[b].data_ptr(), N_LAYER, max_t)
                                             for b in range(self.B)])
        self.h = ctypes.c_void_p()
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

    def generate(self, prompt, prompt_len, n_steps: int, out, stream: int = 0) -> None:
        """prompt: int32 [B][P]; prompt_len: int32 [B] (1..P); out: int32 [B][>= n_steps+1]."""
        self.lib.check(self.lib.gpt2_b200_batch_generate(
            self.h, prompt.data_ptr(), prompt.stride(0), prompt_len.data_ptr(), n_steps,
            out.data_ptr(), out.stride(0), 0, stream), "gpt2_b200_batch_generate")

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
        if out.shape[1] <= n_steps < out.stride(0):  # a view whose rows end early: the library sees the stride alone
            raise ValueError("generate: out is too narrow")
        self.lib.check(self.lib.gpt2_b200_beam_generate(
            self.h, prompt.data_ptr(), prompt.stride(0), _vector(what, prompt_len, i32, self.B, at), n_steps, eos, out.data_ptr(),
            out.stride(0), _vector(what, score, f32, rows, at) if score is not None else None, stream), "gpt2_b200_beam_generate")

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
