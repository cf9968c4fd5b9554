"""ctypes binding of libbq.so (include/bq.h) over torch device tensors.

torch supplies device memory and the current HIP stream; every computation runs
in libbq's HIP kernels.  There is no fallback: if libbq.so is missing or the
GPU is absent, calls raise.

Host-side mirror of the reference's launchers (engine/src/bruce.cu):
    gemv                  launch_gemv            :5624
    verify_fused          launch_verify_fused    :7141
    q6_verify_fused       launch_q6_verify_fused :7231
    gemm_q6k_dp           launch_gemm_q6k_dp     :7285
    try_mmq               try_launch_mmq         :7366
    gemm_b / gemm_b_fused launch_gemm_b(_fused)  :7421-7568
    repack_q5k            q5k_prepack_launch     :4832
    repack_q6k(_host)     q6k_repack_host        :4783
    quantize_q8           k_q8_quant / k_q8_rows :518, :1081
    quantize_q8s(_host)   k_bf16_to_q8 / q8k_quant_host :5159, :4843
    gemv_q8s              k_gemm_q8_logits       :4409 (launch_logits_b :7570)
    norm_q8 / add_norm_q8 / resid_q8 / gate_norm_q8 / silu_mul_norm_q8
                          k_norm :541, k_add_norm :556, k_resid :571, k_gate_norm :602,
                          k_silu_mul_norm :622 (and their _rows / _vec4 forms)
"""
import ctypes
import os

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libbq.so")

BQ_OK, BQ_UNSUPPORTED, BQ_EINVAL, BQ_ETOOBIG = 0, 1, 2, 3
TYPE_Q5_K, TYPE_Q6_K = 13, 14
TYPE_F32, TYPE_Q8_0, TYPE_BF16 = 0, 8, 30
Q5K_BYTES, Q6K_BYTES = 176, 210
Q8S_BYTES = 272  # Q8_0 logits head: 8 fp16 scales + 256 int8 per (row, 256 values)

EXPORTS = [
    "bq_init", "bq_strerror", "bq_version", "bq_quantize_q8", "bq_fill_xdh", "bq_gemv",
    "bq_verify_fused", "bq_q6_verify_fused", "bq_gemm_q6k_dp", "bq_gemm_q6k_raw", "bq_try_mmq",
    "bq_gemm_q6k_mma", "bq_gemm_b", "bq_gemm_b_fused", "bq_repack_q5k", "bq_repack_q5k_bytes",
    "bq_repack_q5k_min_bytes", "bq_repack_q6k", "bq_repack_q6k_host", "bq_repack_q6k_bytes",
    "bq_time_next_launch", "bq_gemv_q8_fused", "bq_q8s_bytes", "bq_quantize_q8s",
    "bq_quantize_q8s_host", "bq_gemv_q8s", "bq_norm_q8", "bq_add_norm_q8", "bq_resid_q8",
    "bq_gate_norm_q8", "bq_silu_mul_norm_q8", "bq_gguf_open", "bq_gguf_close", "bq_gguf_n_tensors",
    "bq_gguf_find", "bq_gguf_tensor_info", "bq_gguf_kv_num", "bq_gguf_kv_str", "bq_gguf_read", "bq_gguf_load",
    "bq_gemv_norm_fused", "bq_gate_up_silu", "bq_gemm_workspace_bytes", "bq_gemm_workspace_bytes_cus",
    "bq_gemm_b_fused_noalloc",
    "bq_noalloc_scratch_bytes", "bq_decode_enqueue", "bq_decode_graph_create", "bq_decode_graph_launch",
    "bq_decode_graph_destroy", "bq_kv_page_bytes", "bq_append", "bq_kv_read", "bq_attn_workspace_bytes",
    "bq_attn_prefill_workspace_bytes", "bq_attn_decode", "bq_attn_prefill", "bq_attn_hook", "bq_sample_workspace_bytes", "bq_sample",
]


class BqError(RuntimeError):
    def __init__(self, code, what):
        self.code = code
        super().__init__(f"{what}: {strerror(code)} ({code})")


class Weight(ctypes.Structure):
    """bq_weight == the reference's TensorW {d, dp, dm, type, K, N} (bruce.cu:78)."""
    _fields_ = [("raw", ctypes.c_void_p), ("rep", ctypes.c_void_p), ("rep_min", ctypes.c_void_p),
                ("ggml_type", ctypes.c_uint32), ("K", ctypes.c_int32), ("N", ctypes.c_int32)]


class GgufTensor(ctypes.Structure):
    """bq_gguf_tensor (include/bq.h)."""
    _fields_ = [("name", ctypes.c_char_p), ("suffix", ctypes.c_char_p), ("ne", ctypes.c_uint64 * 4),
                ("offset", ctypes.c_uint64), ("nbytes", ctypes.c_uint64), ("ggml_type", ctypes.c_uint32),
                ("ndim", ctypes.c_uint32), ("block", ctypes.c_int32)]


BLOCK_ATTN, BLOCK_FFN = 0, 1
ATTN_HOOK = ctypes.CFUNCTYPE(None, ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p)


class DecodeBlock(ctypes.Structure):
    """bq_decode_block (include/bq.h): one attention or FFN block of the decode step."""
    _fields_ = [("kind", ctypes.c_int), ("norm_before", ctypes.c_int), ("norm_after", ctypes.c_int),
                ("alpha", ctypes.c_void_p),
                ("qkv", ctypes.POINTER(Weight)), ("n_qkv", ctypes.c_int), ("qkv_out", ctypes.POINTER(ctypes.c_void_p)),
                ("attn_out", ctypes.c_void_p), ("attn_gate", ctypes.c_void_p), ("sgate", ctypes.c_void_p),
                ("n_attn", ctypes.c_int), ("o", ctypes.POINTER(Weight)),
                ("gate", ctypes.POINTER(Weight)), ("up", ctypes.POINTER(Weight)),
                ("s_gate", ctypes.c_void_p), ("s_up", ctypes.c_void_p), ("down", ctypes.POINTER(Weight)),
                ("n_ff", ctypes.c_int)]


class DecodeStep(ctypes.Structure):
    """bq_decode_step (include/bq.h): the per-token decode launch sequence."""
    _fields_ = [("n_blocks", ctypes.c_int), ("blocks", ctypes.POINTER(DecodeBlock)), ("n_embd", ctypes.c_int),
                ("fold", ctypes.c_int), ("x", ctypes.c_void_p), ("input_h", ctypes.c_void_p),
                ("xq", ctypes.c_void_p), ("xd", ctypes.c_void_p), ("xsum", ctypes.c_void_p),
                ("proj", ctypes.c_void_p), ("ffn_g", ctypes.c_void_p), ("ffn_u", ctypes.c_void_p),
                ("attention", ATTN_HOOK), ("user", ctypes.c_void_p),
                ("head_q8s", ctypes.c_void_p), ("head_rs", ctypes.c_void_p), ("head", ctypes.POINTER(Weight)),
                ("vocab", ctypes.c_int), ("logits", ctypes.c_void_p), ("rows", ctypes.c_int),
                ("x_alt", ctypes.c_void_p), ("xdh", ctypes.c_void_p), ("work", ctypes.c_void_p),
                ("work_bytes", ctypes.c_size_t)]


class KvCacheStruct(ctypes.Structure):
    """bq_kv_cache (include/bq.h): the paged key-value cache."""
    _fields_ = [("pages", ctypes.c_void_p), ("table", ctypes.c_void_p), ("type", ctypes.c_int),
                ("kv_heads", ctypes.c_int), ("head_dim", ctypes.c_int), ("page_tokens", ctypes.c_int),
                ("n_pages", ctypes.c_int), ("n_seq", ctypes.c_int), ("max_pages", ctypes.c_int)]


class AppendArgs(ctypes.Structure):
    """bq_append_args (include/bq.h)."""
    _fields_ = [("q", ctypes.c_void_p), ("k", ctypes.c_void_p), ("v", ctypes.c_void_p),
                ("ldq", ctypes.c_int64), ("ldk", ctypes.c_int64), ("ldv", ctypes.c_int64),
                ("rows", ctypes.c_int), ("q_heads", ctypes.c_int), ("pos", ctypes.c_void_p), ("seq", ctypes.c_void_p),
                ("q_weight", ctypes.c_void_p), ("k_weight", ctypes.c_void_p), ("eps", ctypes.c_float),
                ("rope", ctypes.c_void_p), ("rot", ctypes.c_int), ("n_pos", ctypes.c_int),
                ("interleaved", ctypes.c_int), ("q_out", ctypes.c_void_p), ("q_type", ctypes.c_int)]


class AttnArgs(ctypes.Structure):
    """bq_attn_args (include/bq.h)."""
    _fields_ = [("q", ctypes.c_void_p), ("out", ctypes.c_void_p), ("q_type", ctypes.c_int), ("out_type", ctypes.c_int),
                ("ldq", ctypes.c_int64), ("ldo", ctypes.c_int64), ("q_heads", ctypes.c_int), ("n_rows", ctypes.c_int),
                ("rows", ctypes.c_int), ("row0", ctypes.c_void_p), ("kv_len", ctypes.c_void_p),
                ("max_len", ctypes.c_int), ("scale", ctypes.c_float), ("window", ctypes.c_int), ("sinks", ctypes.c_int),
                ("work", ctypes.c_void_p), ("work_bytes", ctypes.c_size_t)]


class AttnBlock(ctypes.Structure):
    """bq_attn_block (include/bq.h): what the attention hook runs for one block of the step."""
    _fields_ = [("kv", ctypes.POINTER(KvCacheStruct)), ("append", ctypes.POINTER(AppendArgs)),
                ("attn", ctypes.POINTER(AttnArgs)), ("prefill", ctypes.c_int)]


class AttnPlanStruct(ctypes.Structure):
    """bq_attn_plan (include/bq.h)."""
    _fields_ = [("n_blocks", ctypes.c_int), ("blocks", ctypes.POINTER(AttnBlock)), ("status", ctypes.c_int)]


_lib = None


def load(path=LIB_PATH):
    """Load libbq.so (raises if it is not built).  Imports torch first so the
    HIP runtime libbq links against is torch's own."""
    global _lib
    if _lib is not None:
        return _lib
    import torch  # noqa: F401  (one HIP runtime per process)
    if not os.path.exists(path):
        raise FileNotFoundError(f"{path} is not built: run __graft_entry__.build()")
    L = ctypes.CDLL(path)
    P, I, S = ctypes.c_void_p, ctypes.c_int, ctypes.c_size_t
    WP = ctypes.POINTER(Weight)
    sig = {
        "bq_init": (I, []),
        "bq_strerror": (ctypes.c_char_p, [I]),
        "bq_version": (ctypes.c_char_p, []),
        "bq_quantize_q8": (I, [P, I, I, P, P, P, P, P]),
        "bq_fill_xdh": (I, [P, P, I, P, P]),
        "bq_gemv": (I, [P, WP, P, P, P, P]),
        "bq_verify_fused": (I, [P, P, I, I, P, P, P, I, P]),
        "bq_q6_verify_fused": (I, [P, P, I, I, P, P, I, P]),
        "bq_gemm_q6k_dp": (I, [P, WP, I, P, P, I, P]),
        "bq_gemm_q6k_raw": (I, [P, WP, I, P, P, I, P]),
        "bq_gemm_workspace_bytes": (S, [I, I, I]),
        "bq_gemm_workspace_bytes_cus": (S, [I, I, I, I]),
        "bq_try_mmq": (I, [P, P, I, I, P, P, P, P, P, S, P]),
        "bq_gemm_q6k_mma": (I, [P, WP, I, P, P, P, S, P]),
        "bq_gemm_b": (I, [P, WP, I, P, P, P, P, P, S, P]),
        "bq_gemm_b_fused": (I, [P, P, I, I, P, P, P, P, P, S, P]),
        "bq_gemm_b_fused_noalloc": (I, [P, P, I, I, P, P, P, P]),
        "bq_decode_enqueue": (I, [ctypes.POINTER(DecodeStep), P]),
        "bq_decode_graph_create": (I, [ctypes.POINTER(DecodeStep), P, ctypes.POINTER(P)]),
        "bq_decode_graph_launch": (I, [P, P]),
        "bq_decode_graph_destroy": (None, [P]),
        "bq_noalloc_scratch_bytes": (S, []),
        "bq_repack_q5k": (I, [P, I, I, P, P, P]),
        "bq_repack_q5k_bytes": (S, [I, I]),
        "bq_repack_q5k_min_bytes": (S, [I, I]),
        "bq_repack_q6k": (I, [P, I, I, P, P]),
        "bq_repack_q6k_host": (I, [P, I, I, P]),
        "bq_repack_q6k_bytes": (S, [I, I]),
        "bq_time_next_launch": (I, [P, P]),
        "bq_gemv_q8_fused": (I, [P, P, I, P, P, P, P, P]),
        "bq_gemv_norm_fused": (I, [P, P, I, I, P, P, P, P, P, P, P, P, P]),
        "bq_gate_up_silu": (I, [P, WP, WP, P, P, P, P, P, P]),
        "bq_q8s_bytes": (S, [I, I]),
        "bq_quantize_q8s": (I, [P, I, I, P, P]),
        "bq_quantize_q8s_host": (I, [P, I, I, P]),
        "bq_gemv_q8s": (I, [P, P, P, P, I, I, I, P, P]),
        "bq_norm_q8": (I, [P, P, I, I, P, P, P, P]),
        "bq_add_norm_q8": (I, [P, P, I, I, P, P, P, P]),
        "bq_resid_q8": (I, [P, P, P, I, I, P, P, P, P]),
        "bq_gate_norm_q8": (I, [P, P, P, P, I, I, P, P, P, P]),
        "bq_silu_mul_norm_q8": (I, [P, P, P, P, P, I, I, P, P, P, P]),
        "bq_gguf_open": (I, [ctypes.c_char_p, ctypes.POINTER(P)]),
        "bq_gguf_close": (None, [P]),
        "bq_gguf_n_tensors": (ctypes.c_int64, [P]),
        "bq_gguf_find": (ctypes.c_int64, [P, ctypes.c_char_p]),
        "bq_gguf_tensor_info": (I, [P, ctypes.c_int64, ctypes.POINTER(GgufTensor)]),
        "bq_gguf_kv_num": (I, [P, ctypes.c_char_p, ctypes.POINTER(ctypes.c_double)]),
        "bq_gguf_kv_str": (I, [P, ctypes.c_char_p, ctypes.POINTER(ctypes.c_char_p)]),
        "bq_gguf_read": (I, [P, ctypes.c_int64, P, S, ctypes.c_uint64]),
        "bq_gguf_load": (I, [P, ctypes.c_int64, P, P, P, WP, P]),
        "bq_kv_page_bytes": (S, [I, I, I, I]),
        "bq_append": (I, [P, P, P]),
        "bq_kv_read": (I, [P, P, P, I, P, P, P]),
        "bq_attn_workspace_bytes": (S, [I, I, I, I, I, I]),
        "bq_attn_prefill_workspace_bytes": (S, [I] * 8),
        "bq_attn_decode": (I, [P, P, P]),
        "bq_attn_prefill": (I, [P, P, P]),
        "bq_attn_hook": (None, [P, I, P]),
        "bq_sample_workspace_bytes": (S, [I, I]),
        "bq_sample": (I, [P, ctypes.c_int64, I, I, P, P, P, P, P, P, P, S, P]),
    }
    for name, (res, args) in sig.items():
        f = getattr(L, name)
        f.restype = res
        f.argtypes = args
    _lib = L
    return L


def strerror(code):
    return load().bq_strerror(code).decode()


def _check(code, what):
    if code != BQ_OK:
        raise BqError(code, what)
    return code


def _ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream():
    import torch
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _need_gpu(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("libbq entry points take device tensors")


def make_weight(raw=None, ggml_type=TYPE_Q5_K, K=0, N=0, rep=None, rep_min=None):
    """Build a bq_weight; the tensors must stay alive while it is used."""
    w = Weight(_ptr(raw).value if raw is not None else None,
               _ptr(rep).value if rep is not None else None,
               _ptr(rep_min).value if rep_min is not None else None, ggml_type, K, N)
    w._keep = (raw, rep, rep_min)
    return w


# ---------------------------------------------------------------- quantizer
def quantize_q8(x, with_xdh=False):
    """x fp32 [rows, K] (device) -> xq int8 [rows,K], xd fp32 [rows,K/32], xsum int32, (xdh)."""
    import torch
    _need_gpu(x)
    x = x.contiguous()
    rows, K = x.shape
    xq = torch.empty((rows, K), dtype=torch.int8, device=x.device)
    xd = torch.empty((rows, K // 32), dtype=torch.float32, device=x.device)
    xs = torch.empty((rows, K // 32), dtype=torch.int32, device=x.device)
    xdh = torch.empty((rows, K // 32), dtype=torch.int16, device=x.device) if with_xdh else None
    _check(load().bq_quantize_q8(_ptr(x), rows, K, _ptr(xq), _ptr(xd), _ptr(xs), _ptr(xdh), _stream()),
           "bq_quantize_q8")
    return (xq, xd, xs, xdh) if with_xdh else (xq, xd, xs)


def fill_xdh(xd, xsum, out=None):
    import torch
    if out is None:
        out = torch.empty(xd.shape, dtype=torch.int16, device=xd.device)
    _check(load().bq_fill_xdh(_ptr(xd), _ptr(xsum), xd.numel(), _ptr(out), _stream()), "bq_fill_xdh")
    return out


# ---------------------------------------------------------------- GEMV / verify
def gemv(y, w, xq, xd, xsum):
    _check(load().bq_gemv(_ptr(y), ctypes.byref(w), _ptr(xq), _ptr(xd), _ptr(xsum), _stream()), "bq_gemv")
    return y


def _arrays(ys, ws):
    n = len(ws)
    yarr = (ctypes.c_void_p * n)(*[y.data_ptr() for y in ys])
    warr = (ctypes.POINTER(Weight) * n)(*[ctypes.pointer(w) for w in ws])
    return yarr, warr


def verify_fused(ys, ws, rows, xq, xd, xsum, xoff=0):
    """Returns the raw code (BQ_UNSUPPORTED means nothing ran, as the reference's false)."""
    yarr, warr = _arrays(ys, ws)
    r = load().bq_verify_fused(yarr, warr, len(ws), rows, _ptr(xq), _ptr(xd), _ptr(xsum), xoff, _stream())
    if r not in (BQ_OK, BQ_UNSUPPORTED):
        raise BqError(r, "bq_verify_fused")
    return r


def gemv_q8_fused(ys, ws, x, xq=None, xd=None, xsum=None):
    """Quantize the fp32 row x and run the GEMV over every part in one launch;
    xq/xd/xsum (all or none) receive the q8 row."""
    yarr, warr = _arrays(ys, ws)
    r = load().bq_gemv_q8_fused(yarr, warr, len(ws), _ptr(x), _ptr(xq), _ptr(xd), _ptr(xsum), _stream())
    if r not in (BQ_OK, BQ_UNSUPPORTED):
        raise BqError(r, "bq_gemv_q8_fused")
    return r


OPS = {"norm": 0, "add": 1, "resid": 2, "gate": 3, "silu": 4}


def gemv_norm_fused(ys, ws, op, a, b=None, c=None, d=None, out=None, q8=None):
    """q8 producer (op as norm_q8: norm a; add a+b; resid x=a, upd=b, alpha=c;
    gate aout=a, gate=b, sg=c; silu g=a, u=b, sg=c, su=d) and the GEMV of its
    row over every part, one launch.  out receives the produced fp32 row, q8 =
    (xq, xd, xsum) its q8 row.  Returns the raw code (BQ_UNSUPPORTED: nothing ran)."""
    _need_gpu(a, b, c, d, out)
    yarr, warr = _arrays(ys, ws)
    xq, xd, xs = q8 if q8 is not None else (None, None, None)
    r = load().bq_gemv_norm_fused(yarr, warr, len(ws), OPS[op], _ptr(out), _ptr(a), _ptr(b), _ptr(c), _ptr(d),
                                  _ptr(xq), _ptr(xd), _ptr(xs), _stream())
    if r not in (BQ_OK, BQ_UNSUPPORTED):
        raise BqError(r, "bq_gemv_norm_fused")
    return r


def gate_up_silu(h, wg, wu, sg, su, xq, xd, xsum=None):
    """h = silu(g * sg) * u * su with g = wg x, u = wu x for one q8 row x, one launch."""
    _need_gpu(h, sg, su, xq, xd, xsum)
    _check(load().bq_gate_up_silu(_ptr(h), ctypes.byref(wg), ctypes.byref(wu), _ptr(sg), _ptr(su), _ptr(xq),
                                  _ptr(xd), _ptr(xsum), _stream()), "bq_gate_up_silu")
    return h


def q6_verify_fused(ys, ws, rows, xq, xd, xoff=0):
    yarr, warr = _arrays(ys, ws)
    r = load().bq_q6_verify_fused(yarr, warr, len(ws), rows, _ptr(xq), _ptr(xd), xoff, _stream())
    if r not in (BQ_OK, BQ_UNSUPPORTED):
        raise BqError(r, "bq_q6_verify_fused")
    return r


def gemm_q6k_dp(y, w, rows, xq, xd, xoff=0):
    return _check(load().bq_gemm_q6k_dp(_ptr(y), ctypes.byref(w), rows, _ptr(xq), _ptr(xd), xoff, _stream()),
                  "bq_gemm_q6k_dp")


def gemm_q6k_raw(y, w, rows, xq, xd, xoff=0):
    return _check(load().bq_gemm_q6k_raw(_ptr(y), ctypes.byref(w), rows, _ptr(xq), _ptr(xd), xoff, _stream()),
                  "bq_gemm_q6k_raw")


# ---------------------------------------------------------------- prefill GEMM
def workspace_bytes(rows, K, n_total):
    """bq_gemm_workspace_bytes: K-split workspace that allows the full split."""
    return int(load().bq_gemm_workspace_bytes(rows, K, n_total))


def workspace(rows, K, n_total, device="cuda"):
    """A K-split workspace for GEMMs of rows x (n_total = sum N) x K (None if
    such a launch never splits).  Allocated by torch: libbq itself allocates
    nothing."""
    import torch
    n = workspace_bytes(rows, K, n_total)
    return torch.empty(n // 4, dtype=torch.float32, device=device) if n else None


_ws_cache = {}  # (device, stream) -> the largest workspace handed out there so far


def _work(work, rows, K, n_total):
    """work="auto": a workspace sized for the full split, one per (device,
    stream) reused by every call there (calls on one stream are ordered, so
    they can share it) and grown when a shape needs more; None: no split; a
    tensor: used as given.  Returns (pointer, bytes, tensor kept alive by the
    caller)."""
    if isinstance(work, str):
        assert work == "auto"
        import torch
        n = workspace_bytes(rows, K, n_total)
        if n == 0:
            return None, 0, None
        key = (torch.cuda.current_device(), torch.cuda.current_stream().cuda_stream)
        work = _ws_cache.get(key)
        if work is None or work.numel() * 4 < n:
            work = torch.empty(n // 4, dtype=torch.float32, device="cuda")
            _ws_cache[key] = work
    if work is None:
        return None, 0, None
    return _ptr(work), work.numel() * work.element_size(), work


def try_mmq(ys, ws, rows, xq, xd, xsum, xdh=None, work="auto"):
    wp, wb, keep = _work(work, rows, ws[0].K, sum(w.N for w in ws))
    yarr, warr = _arrays(ys, ws)
    r = load().bq_try_mmq(yarr, warr, len(ws), rows, _ptr(xq), _ptr(xd), _ptr(xsum), _ptr(xdh), wp, wb, _stream())
    if r not in (BQ_OK, BQ_UNSUPPORTED):
        raise BqError(r, "bq_try_mmq")
    return r


def gemm_q6k_mma(y, w, rows, xq, xd, work="auto"):
    wp, wb, keep = _work(work, rows, w.K, w.N)
    return _check(load().bq_gemm_q6k_mma(_ptr(y), ctypes.byref(w), rows, _ptr(xq), _ptr(xd), wp, wb, _stream()),
                  "bq_gemm_q6k_mma")


def gemm_b(y, w, rows, xq, xd, xsum, xdh=None, work="auto"):
    wp, wb, keep = _work(work, rows, w.K, w.N)
    return _check(load().bq_gemm_b(_ptr(y), ctypes.byref(w), rows, _ptr(xq), _ptr(xd), _ptr(xsum),
                                   _ptr(xdh), wp, wb, _stream()), "bq_gemm_b")


def gemm_b_fused(ys, ws, rows, xq, xd, xsum, xdh=None, work="auto"):
    wp, wb, keep = _work(work, rows, ws[0].K, sum(w.N for w in ws))
    yarr, warr = _arrays(ys, ws)
    return _check(load().bq_gemm_b_fused(yarr, warr, len(ws), rows, _ptr(xq), _ptr(xd), _ptr(xsum),
                                         _ptr(xdh), wp, wb, _stream()), "bq_gemm_b_fused")


# ---------------------------------------------------------------- repacks
def repack_q5k(raw, K, N):
    """raw uint8 device [N, K/256*176] -> (W144 uint8 [K/128, N, 144], Dm int16 [N, K/32])."""
    import torch
    w144 = torch.empty((K // 128, N, 144), dtype=torch.uint8, device=raw.device)
    dm = torch.empty((N, K // 32), dtype=torch.int16, device=raw.device)
    _check(load().bq_repack_q5k(_ptr(raw), K, N, _ptr(w144), _ptr(dm), _stream()), "bq_repack_q5k")
    return w144, dm


def repack_q6k(raw, K, N):
    import torch
    out = torch.empty((N, K // 128, 160), dtype=torch.uint8, device=raw.device)
    _check(load().bq_repack_q6k(_ptr(raw), K, N, _ptr(out), _stream()), "bq_repack_q6k")
    return out


def repack_q6k_host(raw_np, K, N):
    """Host twin on numpy arrays (no device)."""
    import numpy as np
    raw_np = np.ascontiguousarray(raw_np, np.uint8)
    out = np.empty((N, K // 128, 160), np.uint8)
    _check(load().bq_repack_q6k_host(raw_np.ctypes.data_as(ctypes.c_void_p), K, N,
                                     out.ctypes.data_as(ctypes.c_void_p)), "bq_repack_q6k_host")
    return out


# ---------------------------------------------------------------- Q8_0 logits head
def quantize_q8s(w_bf16, K, N):
    """bf16 bit patterns (int16/uint16 device tensor [N, K]) -> Q8S uint8 [N, K/256*272]."""
    import torch
    _need_gpu(w_bf16)
    out = torch.empty((N, K // 256 * Q8S_BYTES), dtype=torch.uint8, device=w_bf16.device)
    _check(load().bq_quantize_q8s(_ptr(w_bf16.contiguous()), K, N, _ptr(out), _stream()), "bq_quantize_q8s")
    return out


def quantize_q8s_host(w_bf16_np, K, N):
    """Host twin on a numpy uint16 array (no device)."""
    import numpy as np
    w = np.ascontiguousarray(w_bf16_np, np.uint16)
    out = np.empty((N, K // 256 * Q8S_BYTES), np.uint8)
    _check(load().bq_quantize_q8s_host(w.ctypes.data_as(ctypes.c_void_p), K, N,
                                       out.ctypes.data_as(ctypes.c_void_p)), "bq_quantize_q8s_host")
    return out


def gemv_q8s(y, w, xq, xd, K, N, rows, rs=None):
    """y fp32 [rows, N] = Q8S w [N, K] x q8 rows (xq [rows, K], xd [rows, K/32]), times rs[N]."""
    _need_gpu(y, w, xq, xd, rs)
    r = load().bq_gemv_q8s(_ptr(y), _ptr(w), _ptr(xq), _ptr(xd), K, N, rows, _ptr(rs), _stream())
    if r not in (BQ_OK, BQ_UNSUPPORTED):
        raise BqError(r, "bq_gemv_q8s")
    return r


# ---------------------------------------------------------------- q8 producers
def _q8_out(rows, n, device):
    import torch
    return (torch.empty((rows, n), dtype=torch.int8, device=device),
            torch.empty((rows, n // 32), dtype=torch.float32, device=device),
            torch.empty((rows, n // 32), dtype=torch.int32, device=device))


def norm_q8(op, rows, n, out=None, a=None, b=None, c=None, d=None, q8=None):
    """op in {"norm", "add", "resid", "gate", "silu"}; returns (out, (xq, xd, xsum)).
    norm: out = norm(a); add: a = norm(a + b) in place; resid: a = norm(norm(a) +
    (norm(b) - norm(a))*c) in place; gate: out = norm(a / (1 + exp(-b*c)));
    silu: out = norm(silu(a*c) * b * d)."""
    _need_gpu(out, a, b, c, d)
    if q8 is None:
        q8 = _q8_out(rows, n, a.device)
    xq, xd, xs = q8
    L = load()
    S = _stream()
    if op == "norm":
        r = L.bq_norm_q8(_ptr(out), _ptr(a), rows, n, _ptr(xq), _ptr(xd), _ptr(xs), S)
    elif op == "add":
        r = L.bq_add_norm_q8(_ptr(a), _ptr(b), rows, n, _ptr(xq), _ptr(xd), _ptr(xs), S)
    elif op == "resid":
        r = L.bq_resid_q8(_ptr(a), _ptr(b), _ptr(c), rows, n, _ptr(xq), _ptr(xd), _ptr(xs), S)
    elif op == "gate":
        r = L.bq_gate_norm_q8(_ptr(out), _ptr(a), _ptr(b), _ptr(c), rows, n, _ptr(xq), _ptr(xd), _ptr(xs), S)
    elif op == "silu":
        r = L.bq_silu_mul_norm_q8(_ptr(out), _ptr(a), _ptr(b), _ptr(c), _ptr(d), rows, n, _ptr(xq), _ptr(xd),
                                  _ptr(xs), S)
    else:
        raise ValueError(op)
    if r not in (BQ_OK, BQ_UNSUPPORTED):
        raise BqError(r, f"norm_q8({op})")
    return r, q8


# ---------------------------------------------------------------- GGUF
class Gguf:
    """GGUF v3 file opened by libbq's reader (bq_gguf_*)."""

    def __init__(self, path):
        self._h = ctypes.c_void_p()
        _check(load().bq_gguf_open(os.fsencode(path), ctypes.byref(self._h)), f"bq_gguf_open({path})")

    def close(self):
        if self._h:
            load().bq_gguf_close(self._h)
            self._h = ctypes.c_void_p()

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __len__(self):
        return load().bq_gguf_n_tensors(self._h)

    def find(self, name):
        return load().bq_gguf_find(self._h, name.encode())

    def tensor(self, i):
        t = GgufTensor()
        _check(load().bq_gguf_tensor_info(self._h, i, ctypes.byref(t)), "bq_gguf_tensor_info")
        return {"name": t.name.decode(errors="replace"), "suffix": t.suffix.decode(errors="replace"), "ne": list(t.ne)[:t.ndim],
                "offset": t.offset, "nbytes": t.nbytes, "type": t.ggml_type, "ndim": t.ndim, "block": t.block}

    def kv_num(self, key):
        v = ctypes.c_double()
        r = load().bq_gguf_kv_num(self._h, key.encode(), ctypes.byref(v))
        return v.value if r == BQ_OK else None

    def kv_str(self, key):
        v = ctypes.c_char_p()
        r = load().bq_gguf_kv_str(self._h, key.encode(), ctypes.byref(v))
        return v.value.decode(errors="replace") if r == BQ_OK else None

    def read(self, i, n=None, off=0):
        import numpy as np
        nb = self.tensor(i)["nbytes"]
        n = nb - off if n is None else n
        out = np.empty(n, np.uint8)
        _check(load().bq_gguf_read(self._h, i, out.ctypes.data_as(ctypes.c_void_p), n, off), "bq_gguf_read")
        return out

    def load(self, i, raw, rep=None, rep_min=None):
        """Stream tensor i into device tensor `raw` (+ repack into rep / rep_min); returns a Weight."""
        w = Weight()
        r = load().bq_gguf_load(self._h, i, _ptr(raw), _ptr(rep), _ptr(rep_min), ctypes.byref(w), _stream())
        if r != BQ_OK:
            raise BqError(r, "bq_gguf_load")
        w._keep = (raw, rep, rep_min)
        return w


# ---------------------------------------------------------------- decode step
def decode_enqueue(step):
    return _check(load().bq_decode_enqueue(ctypes.byref(step), _stream()), "bq_decode_enqueue")


class DecodeGraph:
    """bq_decode_graph: the captured decode step; launch() replays one token."""

    def __init__(self, step):
        self.step = step   # keeps the ctypes structures alive
        h = ctypes.c_void_p()
        _check(load().bq_decode_graph_create(ctypes.byref(step), _stream(), ctypes.byref(h)),
               "bq_decode_graph_create")
        self.h = h

    def launch(self):
        return _check(load().bq_decode_graph_launch(self.h, _stream()), "bq_decode_graph_launch")

    def close(self):
        if self.h:
            load().bq_decode_graph_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


# ---------------------------------------------------------------- serving operators
# the current device, and a device's current stream as a number (torch.cuda's own functions check and build
# more, and a call of an operator takes a few microseconds)
_current = _raw_stream = None


def _bind_device():
    global _current, _raw_stream
    if _current is None:
        import torch
        _current = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", lambda d: torch.cuda.current_stream(d).cuda_stream)


def _on(device, f, *args):
    """f(*args, stream) on the current stream of a device that is not the current one."""
    import torch
    with torch.cuda.device(device):
        return f(*args, _raw_stream(device))


def _one_device(device, **tensors):
    """ValueError unless every tensor (or None) lies on this device."""
    for what, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{what}: on {device}, not {t.device}")


def _work_of(work, device):
    """A caller's workspace (or None): its bytes have to be there, and on the device."""
    if work is not None and (not work.is_cuda or work.device != device or not work.is_contiguous()):
        raise ValueError(f"work: a contiguous tensor on {device}")
    return work


def _type_of(t, what):
    import torch
    if t.dtype == torch.float32:
        return TYPE_F32
    if t.dtype == torch.bfloat16:
        return TYPE_BF16
    raise TypeError(f"{what}: fp32 or bf16, not {t.dtype}")


def _expect(t, dtype, shape, what):
    """A contiguous device tensor of this dtype and shape (or None)."""
    if t is None:
        return None
    if not t.is_cuda or t.dtype != dtype or tuple(t.shape) != tuple(shape) or not t.is_contiguous():
        raise ValueError(f"{what}: a contiguous device tensor {dtype} {tuple(shape)}, not {t.dtype} {tuple(t.shape)}")
    return t


def _rows_ld(t, width, what):
    """Row stride of a [rows, width] device tensor whose rows are contiguous."""
    if not t.is_cuda or t.dim() != 2 or t.shape[1] != width or (width > 1 and t.stride(1) != 1):
        raise ValueError(f"{what}: device rows of {width} contiguous values, not {tuple(t.shape)}")
    return t.stride(0) if t.shape[0] > 1 else max(width, t.stride(0))


KV_TYPES = {"bf16": TYPE_BF16, "q8": TYPE_Q8_0}


def kv_page_bytes(kv_type, kv_heads, head_dim, page_tokens):
    n = int(load().bq_kv_page_bytes(KV_TYPES[kv_type], kv_heads, head_dim, page_tokens))
    if n == 0:
        raise BqError(BQ_UNSUPPORTED, "bq_kv_page_bytes")
    return n


def rope_table(n_pos, rot, base=10000.0, device="cuda"):
    """fp32 [n_pos, rot]: cosines, then sines, of pos * base^(-2 i / rot), formed in 64 bits."""
    import torch
    i = torch.arange(rot // 2, dtype=torch.float64, device=device)
    a = torch.arange(n_pos, dtype=torch.float64, device=device)[:, None] * base ** (-2.0 * i / rot)
    return torch.cat([a.cos(), a.sin()], 1).float().contiguous()


class KvCache:
    """The paged key-value cache: pages uint8 [n_pages, kv_page_bytes], table int32 [n_seq, max_pages]."""

    def __init__(self, pages, table, kv_type, kv_heads, head_dim, page_tokens):
        import torch
        n = kv_page_bytes(kv_type, kv_heads, head_dim, page_tokens)
        _expect(pages, torch.uint8, (pages.shape[0], n), "pages")
        _expect(table, torch.int32, (table.shape[0], table.shape[1]), "table")
        _one_device(pages.device, table=table)
        self.pages, self.table, self.kv_heads, self.head_dim = pages, table, kv_heads, head_dim
        self.struct = KvCacheStruct(_ptr(pages), _ptr(table), KV_TYPES[kv_type], kv_heads, head_dim, page_tokens,
                                    pages.shape[0], table.shape[0], table.shape[1])
        self.ref = ctypes.byref(self.struct)
        self._read, self.device = load().bq_kv_read, pages.device.index
        _bind_device()

    @classmethod
    def empty(cls, n_pages, table, kv_type, kv_heads, head_dim, page_tokens, device="cuda"):
        """With pages of its own."""
        import torch
        n = kv_page_bytes(kv_type, kv_heads, head_dim, page_tokens)
        return cls(torch.zeros((n_pages, n), dtype=torch.uint8, device=device), table, kv_type, kv_heads, head_dim,
                   page_tokens)

    def read(self, pos, k=None, v=None, seq=None):
        """K and / or V of tokens pos (int32 [rows]) of sequences seq into bf16 [rows, kv_heads * head_dim]."""
        import torch
        rows = pos.shape[0]
        for t, what in ((pos, "pos"), (seq, "seq")):
            _expect(t, torch.int32, (rows,), what)
        for t, what in ((k, "k"), (v, "v")):
            _expect(t, torch.bfloat16, (rows, self.kv_heads * self.head_dim), what)
        _one_device(self.pages.device, pos=pos, seq=seq, k=k, v=v)
        args, d = (self.ref, _ptr(seq), _ptr(pos), rows, _ptr(k), _ptr(v)), self.device
        return _check(self._read(*args, _raw_stream(d)) if _current() == d else _on(d, self._read, *args), "bq_kv_read")


class Append:
    """bq_append over fixed buffers: q [rows, q_heads * D], k and v [rows, kv_heads * D] fp32 (rows may be
    strided), pos and seq int32 [rows], q_out fp32 or bf16 [rows, q_heads * D]; rope fp32 [n_pos, rot] as from
    rope_table (None: no rotation, positions below n_pos)."""

    def __init__(self, kv, q, k, v, pos, q_out, seq=None, q_weight=None, k_weight=None, eps=1e-6, rope=None,
                 n_pos=None, interleaved=False):
        import torch
        rows, D = pos.shape[0], kv.head_dim
        _expect(pos, torch.int32, (rows,), "pos")
        _expect(seq, torch.int32, (rows,), "seq")
        for t, what in ((q_weight, "q_weight"), (k_weight, "k_weight")):
            _expect(t, torch.float32, (D,), what)
        if rope is not None:
            _expect(rope, torch.float32, tuple(rope.shape), "rope")
        width = q_out.shape[1]
        _expect(q_out, q_out.dtype, (rows, width), "q_out")
        if width % D:
            raise ValueError("q_out: whole heads")
        for t, what in ((q, "q"), (k, "k"), (v, "v")):
            if t.dtype != torch.float32 or t.shape[0] != rows:
                raise ValueError(f"{what}: fp32 rows, as many as pos has")
        ld = [_rows_ld(q, width, "q")] + [_rows_ld(t, kv.kv_heads * D, "k, v") for t in (k, v)]
        _one_device(kv.pages.device, q=q, k=k, v=v, pos=pos, seq=seq, q_weight=q_weight, k_weight=k_weight, rope=rope, q_out=q_out)
        rot = 0 if rope is None else rope.shape[1]
        if n_pos is None:
            n_pos = (1 << 31) - 1 if rope is None else rope.shape[0]
        elif rope is not None and n_pos > rope.shape[0]:
            raise ValueError("n_pos: at most the rows of rope")
        self.kv, self._keep = kv, (q, k, v, pos, seq, q_weight, k_weight, rope, q_out)
        self.struct = AppendArgs(_ptr(q), _ptr(k), _ptr(v), *ld, rows, width // D, _ptr(pos), _ptr(seq),
                                 _ptr(q_weight), _ptr(k_weight), eps, _ptr(rope), rot, n_pos, int(interleaved),
                                 _ptr(q_out), _type_of(q_out, "q_out"))
        self._ref, self._run = ctypes.byref(self.struct), load().bq_append

    def run(self):
        kv, d = self.kv.ref, self.kv.device
        return _check(self._run(kv, self._ref, _raw_stream(d)) if _current() == d else _on(d, self._run, kv, self._ref), "bq_append")


class Attention:
    """bq_attn_decode / bq_attn_prefill over fixed buffers: q and out [n_rows, q_heads * D] fp32 or bf16 (rows
    may be strided), kv_len int32 [n_seq].  For prefill() of a batch row0 int32 [n_seq + 1], max_rows the most
    rows a sequence has; for decode() every sequence has n_rows / n_seq rows.  work: a workspace tensor of the
    caller's, "auto" for one of the object's own (its `work`, which other objects may share if their calls are
    ordered), None for none (no split)."""

    def __init__(self, kv, q, out, kv_len, scale=None, window=0, sinks=0, max_len=None, row0=None, max_rows=None,
                 work="auto"):
        import torch
        D, n_seq = kv.head_dim, kv.table.shape[0]
        n_rows, width = q.shape
        if width % D or out.shape != q.shape:
            raise ValueError("q and out: rows of whole heads, alike")
        _expect(kv_len, torch.int32, (n_seq,), "kv_len")
        _expect(row0, torch.int32, (n_seq + 1,), "row0")
        _one_device(kv.pages.device, q=q, out=out, kv_len=kv_len, row0=row0)
        P = kv.struct.page_tokens
        if max_len is None:
            max_len = kv.table.shape[1] * P
        if row0 is not None or n_rows == 0:
            rows = max_rows or n_rows or 1
        else:
            rows = n_rows // n_seq
        L = load()
        if isinstance(work, str):
            # without row0 the object serves decode() and, for one sequence, prefill()
            n = 0
            if row0 is None:
                n = L.bq_attn_workspace_bytes(n_seq, rows, width // D, kv.kv_heads, D, max_len)
            if row0 is not None or n_seq == 1:
                n = max(n, L.bq_attn_prefill_workspace_bytes(kv.struct.type, n_seq, rows, n_rows, width // D,
                                                              kv.kv_heads, D, max_len))
            work = torch.empty(n // 4, dtype=torch.float32, device=q.device) if n else None
        _work_of(work, q.device)
        self.kv, self.work, self._keep = kv, work, (q, out, kv_len, row0)
        self.struct = AttnArgs(_ptr(q), _ptr(out), _type_of(q, "q"), _type_of(out, "out"), _rows_ld(q, width, "q"),
                               _rows_ld(out, width, "out"), width // D, n_rows, rows, _ptr(row0), _ptr(kv_len), max_len,
                               D ** -0.5 if scale is None else scale, window, sinks, _ptr(work),
                               0 if work is None else work.numel() * work.element_size())
        self._ref, self._decode, self._prefill = ctypes.byref(self.struct), L.bq_attn_decode, L.bq_attn_prefill

    def decode(self):
        return self._call(self._decode, "bq_attn_decode")

    def prefill(self):
        return self._call(self._prefill, "bq_attn_prefill")

    def _call(self, f, what):
        kv, d = self.kv.ref, self.kv.device
        return _check(f(kv, self._ref, _raw_stream(d)) if _current() == d else _on(d, f, kv, self._ref), what)


class AttentionPlan:
    """The decode step's attention hook over its blocks: blocks[i] None, or (Append, Attention) of block i.
    install(step) sets step.attention and step.user; check() raises what the hook met."""

    def __init__(self, blocks, prefill=False):
        self._keep = blocks
        P = ctypes.pointer
        self._blocks = (AttnBlock * max(1, len(blocks)))(*[
            AttnBlock() if b is None else AttnBlock(P(b[1].kv.struct), P(b[0].struct), P(b[1].struct), int(prefill))
            for b in blocks])
        self.struct = AttnPlanStruct(len(blocks), self._blocks, BQ_OK)

    def install(self, step):
        step.attention = ctypes.cast(load().bq_attn_hook, ATTN_HOOK)
        step.user = ctypes.addressof(self.struct)
        step._attention_plan = self
        return step

    def check(self):
        code, self.struct.status = self.struct.status, BQ_OK
        return _check(code, "bq_attn_hook")


class Sampler:
    """bq_sample over fixed buffers: logits fp32 [rows, vocab] (rows may be strided), out int32 [rows], u fp32
    [rows] in [0, 1); temperature, top_p, min_p fp32 [rows] and top_k int32 [rows], or None."""

    def __init__(self, logits, out, u, temperature=None, top_k=None, top_p=None, min_p=None, work=None):
        import torch
        rows, vocab = logits.shape
        if logits.dtype != torch.float32:
            raise TypeError("logits: fp32")
        _expect(out, torch.int32, (rows,), "out")
        _expect(top_k, torch.int32, (rows,), "top_k")
        for t, what in ((u, "u"), (temperature, "temperature"), (top_p, "top_p"), (min_p, "min_p")):
            _expect(t, torch.float32, (rows,), what)
        _one_device(logits.device, out=out, u=u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
        L = load()
        if work is None:
            work = torch.empty(int(L.bq_sample_workspace_bytes(rows, vocab)), dtype=torch.uint8, device=logits.device)
        _work_of(work, logits.device)
        ld = _rows_ld(logits, vocab, "logits")
        self._keep = (logits, out, u, temperature, top_k, top_p, min_p, work)
        self._args = (_ptr(logits), ld, rows, vocab, _ptr(temperature), _ptr(top_k), _ptr(top_p), _ptr(min_p), _ptr(u),
                      _ptr(out), _ptr(work), work.numel() * work.element_size())
        self._run, self._device = L.bq_sample, logits.device.index
        _bind_device()

    def run(self):
        d = self._device
        return _check(self._run(*self._args, _raw_stream(d)) if _current() == d else _on(d, self._run, *self._args), "bq_sample")
