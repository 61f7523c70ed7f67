"""torch-tensor front end of the C ABI (plumbing: torch only supplies device memory and the stream).

Every call goes through libmx_attn.so; there is no CPU or PyTorch fallback. Tensors must be CUDA (HIP) float16 with a
unit stride along the feature dimension; row strides are taken from the tensors. The plain case of each entry point
(tensors as documented, no tuning, a decode workspace of the caller's) runs in dooms_amd._native; everything else, and every
refused argument, here.
"""
import contextlib
import ctypes
import importlib
import math
import warnings

import torch

from . import _lib

# Tuning that calls without their own `tuning=` argument pass in their descriptors (see tuning()); None: the library's
# plans.
_default_tuning = None


@contextlib.contextmanager
def tuning(**fields):
    """Within the block, calls that do not pass `tuning=` use an mx_attn_tuning with these fields (decode_splits,
    decode_waves, decode_max_workgroups, prefill_plan); the library's plan for the others."""
    global _default_tuning
    saved = _default_tuning
    _default_tuning = dict(fields)
    try:
        yield
    finally:
        _default_tuning = saved


def _tuning(t):
    return _default_tuning if t is None else t


_ext = None
_bound = None   # the library whose functions the extension holds


class _General:
    """Stands in for an extension that is not built: every call goes the general path."""

    def __getattr__(self, name):
        return lambda *args: None


def _native():
    """dooms_amd._native (csrc/binding.cpp), the plain case of the entry points below in C++: each of its functions
    returns what its namesake here does, a code of the library as an int, or None where the general path has to run.
    Without the extension every call goes that way, some 10 us slower; one built for other headers or another torch is
    refused."""
    global _bound, _ext
    L = _lib.lib()
    if _bound is not L:
        try:
            ext = importlib.import_module("._native", __package__)
        except ModuleNotFoundError:
            warnings.warn("dooms_amd._native is not built (`python -m dooms_amd.build` does): calls take the slower general path",
                          RuntimeWarning, stacklevel=3)
            ext = _General()
        except ImportError as e:
            raise ImportError(f"{e}: build the extension for this torch with `python -m dooms_amd.build`") from e
        else:
            if not hasattr(ext, "bind_paged_more"):
                raise ImportError("dooms_amd._native was built from other sources: build it with `python -m dooms_amd.build`")
            ext.bind(L.mx_attn_abi_version(),
                     tuple(ctypes.sizeof(t) for t in (_lib.MxAttnDesc, _lib.MxAttnRope, _lib.MxLinearDesc, _lib.MxSelfAttnDesc)),
                     *[ctypes.cast(getattr(L, f), ctypes.c_void_p).value for f in (
                         "mx_attn_prefill_ws", "mx_attn_decode", "mx_attn_decode_f32", "mx_attn_decode_rope",
                         "mx_attn_prefill_rope_ws", "mx_linear_call_workspace_bytes", "mx_linear",
                         "mx_self_attention_workspace_bytes", "mx_self_attention")])
            ext.bind_paged(L.mx_attn_abi_version(), tuple(ctypes.sizeof(t) for t in (_lib.MxPagedDesc, _lib.MxPagedRope)),
                           *[ctypes.cast(getattr(L, f), ctypes.c_void_p).value
                             for f in ("mx_paged_store", "mx_paged_decode", "mx_paged_prefill")])
            ext.bind_paged_more(L.mx_attn_abi_version(), tuple(ctypes.sizeof(t) for t in (_lib.MxPagedScales, _lib.MxPagedPrefix)),
                                *[ctypes.cast(getattr(L, f), ctypes.c_void_p).value
                                  for f in ("mx_paged_store_e4m3", "mx_paged_decode_e4m3", "mx_paged_prefill_e4m3",
                                            "mx_paged_decode_shared")])
        _ext = ext   # before _bound: another thread that finds the library bound finds the extension too
        _bound = L
    return _ext


def _result(r):
    if type(r) is int:  # a code of the library other than OK
        _lib.check(r)
    return r


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _rows(t: torch.Tensor, name: str, dtype=torch.float16) -> torch.Tensor:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a device tensor")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if t.dim() != 2 or t.stride(1) != 1:
        raise ValueError(f"{name} must be 2-D [rows][features] with unit feature stride")
    return t


def prefill(q, k_cache, v_cache, *, n_head, n_head_kv, head_dim, p0=0, causal=True, n_kv=None, scale=None,
            out=None, lse=None, want_lse=False, workspace=None, tuning=None):
    """mx_attn_prefill: q [n_q][>= n_head*hd], caches [n_kv][>= n_head_kv*hd]. Returns (out, lse or None).
    workspace: "auto" (sized and zeroed here) or a zeroed uint8 device tensor runs mx_attn_prefill_ws, which takes the
    split-KV kernel for chunks of few rows; None runs mx_attn_prefill."""
    if _tuning(tuning) is None:
        r = _native().prefill(q, k_cache, v_cache, n_head, n_head_kv, head_dim, p0, causal, n_kv, scale, out, lse, want_lse,
                              workspace)
        if r is not None:
            return _result(r)
    _rows(q, "q"), _rows(k_cache, "k_cache"), _rows(v_cache, "v_cache")
    if k_cache.stride(0) != v_cache.stride(0):
        raise ValueError("k_cache and v_cache must share a row stride")
    n_q = q.shape[0]
    if out is None:
        out = torch.empty(n_q, n_head * head_dim, dtype=torch.float16, device=q.device)
    _rows(out, "out")
    if want_lse and lse is None:
        lse = torch.empty(n_q, n_head, dtype=torch.float32, device=q.device)
    if scale is None:
        scale = 1.0 / math.sqrt(head_dim)
    d = _lib.make_desc(n_head, n_head_kv, head_dim, n_q, q.stride(0), k_cache.stride(0), out.stride(0), scale,
                       p0=p0, n_kv=0 if n_kv is None else n_kv, causal=1 if causal else 0, tuning=_tuning(tuning))
    if workspace is None:
        _lib.check(_lib.prefill_raw(d, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(),
                                    lse.data_ptr() if lse is not None else 0, _stream()))
        return out, lse
    if isinstance(workspace, str):
        workspace = new_workspace(_lib.prefill_workspace_bytes(d), q.device)
    _lib.check(_lib.prefill_ws_raw(d, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(),
                                   lse.data_ptr() if lse is not None else 0, workspace.data_ptr(), workspace.numel(),
                                   _stream()))
    return out, lse


def decode_workspace_bytes(*, n_head, n_head_kv, head_dim, n_q, batch, max_kv_len, causal=False) -> int:
    d = _lib.make_desc(n_head, n_head_kv, head_dim, n_q, n_head * head_dim, n_head_kv * head_dim,
                       n_head * head_dim, 1.0, causal=1 if causal else 0)
    return _lib.decode_workspace_bytes(d, batch, max_kv_len)


def new_workspace(nbytes: int, device) -> torch.Tensor:
    """A decode workspace of nbytes (torch's caching allocator aligns it to 512 bytes), zeroed by the library."""
    ws = torch.empty(max(nbytes, 256), dtype=torch.uint8, device=device)
    _lib.check(_lib.decode_workspace_init(ws.data_ptr(), ws.numel(), _stream()))
    return ws


def decode(q, k_caches, v_caches, kv_len, *, n_head, n_head_kv, head_dim, n_q=1, causal=False, scale=None,
           out=None, lse=None, want_lse=False, workspace=None, tuning=None):
    """mx_attn_decode (float16 q) or mx_attn_decode_f32 (float32 q and output): q [batch*n_q][>= n_head*hd];
    k_caches/v_caches lists of [>= kv_len[b]][>= n_head_kv*hd] float16 tensors (entries may repeat); kv_len list of
    ints. Returns (out, lse or None)."""
    if workspace is not None and _tuning(tuning) is None:
        r = _native().decode(q, k_caches, v_caches, kv_len, n_head, n_head_kv, head_dim, n_q, causal, scale, out, lse, want_lse,
                             workspace)
        if r is not None:
            return _result(r)
    batch = len(kv_len)
    if len(k_caches) != batch or len(v_caches) != batch:
        raise ValueError("k_caches, v_caches and kv_len must have one entry per sequence")
    f32 = q.dtype == torch.float32
    _rows(q, "q", q.dtype if f32 else torch.float16)
    kv_stride = k_caches[0].stride(0)
    for t in list(k_caches) + list(v_caches):
        _rows(t, "cache")
        if t.stride(0) != kv_stride:
            raise ValueError("every cache must share one row stride")
    if out is None:
        out = torch.empty(q.shape[0], n_head * head_dim, dtype=q.dtype, device=q.device)
    _rows(out, "out", q.dtype)
    if want_lse and lse is None:
        lse = torch.empty(q.shape[0], n_head, dtype=torch.float32, device=q.device)
    if scale is None:
        scale = 1.0 / math.sqrt(head_dim)
    d = _lib.make_desc(n_head, n_head_kv, head_dim, n_q, q.stride(0), kv_stride, out.stride(0), scale,
                       causal=1 if causal else 0, tuning=_tuning(tuning))
    if workspace is None:
        workspace = new_workspace(_lib.decode_workspace_bytes(d, batch, max(kv_len)), q.device)
    _lib.check((_lib.decode_f32_raw if f32 else _lib.decode_raw)(d, list(kv_len), q.data_ptr(), [t.data_ptr() for t in k_caches],
                               [t.data_ptr() for t in v_caches], out.data_ptr(),
                               lse.data_ptr() if lse is not None else 0, workspace.data_ptr(), workspace.numel(),
                               _stream()))
    return out, lse


def decode_rope(qkv, k_caches, v_caches, kv_len, *, n_head, n_head_kv, head_dim, rope_mode, rope_base=10000.0,
                scale=None, out=None, lse=None, want_lse=False, workspace=None, tuning=None):
    """mx_attn_decode_rope, the fused decode step: qkv f32 [batch][>= (n_head + 2 n_head_kv) hd] holds each sequence's
    new token unrotated (q | k | v); the token goes to position kv_len[b] - 1 of k_caches[b] / v_caches[b] (f16,
    written in place). Returns (out f32 [batch][n_head hd], lse or None)."""
    if workspace is not None and _tuning(tuning) is None:
        r = _native().decode_rope(qkv, k_caches, v_caches, kv_len, n_head, n_head_kv, head_dim, rope_mode, rope_base, scale, out,
                                  lse, want_lse, workspace)
        if r is not None:
            return _result(r)
    batch = len(kv_len)
    if len(k_caches) != batch or len(v_caches) != batch:
        raise ValueError("k_caches, v_caches and kv_len must have one entry per sequence")
    _rows(qkv, "qkv", torch.float32)
    kv_stride = k_caches[0].stride(0)
    for t in list(k_caches) + list(v_caches):
        _rows(t, "cache")
        if t.stride(0) != kv_stride:
            raise ValueError("every cache must share one row stride")
    if out is None:
        out = torch.empty(batch, n_head * head_dim, dtype=torch.float32, device=qkv.device)
    _rows(out, "out", torch.float32)
    if want_lse and lse is None:
        lse = torch.empty(batch, n_head, dtype=torch.float32, device=qkv.device)
    if scale is None:
        scale = 1.0 / math.sqrt(head_dim)
    d = _lib.make_desc(n_head, n_head_kv, head_dim, 1, qkv.stride(0), kv_stride, out.stride(0), scale, causal=0,
                       tuning=_tuning(tuning))
    if workspace is None:
        workspace = new_workspace(_lib.decode_workspace_bytes(d, batch, max(kv_len)), qkv.device)
    _lib.check(_lib.decode_rope_raw(d, rope_mode, rope_base, list(kv_len), qkv.data_ptr(),
                                    [t.data_ptr() for t in k_caches], [t.data_ptr() for t in v_caches],
                                    out.data_ptr(), lse.data_ptr() if lse is not None else 0, workspace.data_ptr(),
                                    workspace.numel(), _stream()))
    return out, lse


def prefill_rope(qkv, k_cache, v_cache, *, n_head, n_head_kv, head_dim, rope_mode, rope_base=10000.0, p0=0,
                 causal=True, n_kv=None, scale=None, out=None, lse=None, want_lse=False, workspace=None,
                 tuning=None):
    """mx_attn_prefill_rope: qkv f32 [n_q][>= (n_head + 2 n_head_kv) hd] unrotated rows at positions p0 ..; their keys
    and values are written (rotated, f16) into rows p0 .. of k_cache / v_cache, then the chunk attends.
    Returns (out f32 [n_q][n_head hd], lse or None). workspace ("auto" or a zeroed uint8 device tensor) runs
    mx_attn_prefill_rope_ws."""
    if _tuning(tuning) is None:
        r = _native().prefill_rope(qkv, k_cache, v_cache, n_head, n_head_kv, head_dim, rope_mode, rope_base, p0, causal, n_kv,
                                   scale, out, lse, want_lse, workspace)
        if r is not None:
            return _result(r)
    _rows(qkv, "qkv", torch.float32), _rows(k_cache, "k_cache"), _rows(v_cache, "v_cache")
    if k_cache.stride(0) != v_cache.stride(0):
        raise ValueError("k_cache and v_cache must share a row stride")
    n_q = qkv.shape[0]
    if out is None:
        out = torch.empty(n_q, n_head * head_dim, dtype=torch.float32, device=qkv.device)
    _rows(out, "out", torch.float32)
    if want_lse and lse is None:
        lse = torch.empty(n_q, n_head, dtype=torch.float32, device=qkv.device)
    if scale is None:
        scale = 1.0 / math.sqrt(head_dim)
    d = _lib.make_desc(n_head, n_head_kv, head_dim, n_q, qkv.stride(0), k_cache.stride(0), out.stride(0), scale,
                       p0=p0, n_kv=0 if n_kv is None else n_kv, causal=1 if causal else 0, tuning=_tuning(tuning))
    if workspace is None:
        _lib.check(_lib.prefill_rope_raw(d, rope_mode, rope_base, qkv.data_ptr(), k_cache.data_ptr(),
                                         v_cache.data_ptr(), out.data_ptr(), lse.data_ptr() if lse is not None else 0,
                                         _stream()))
        return out, lse
    if isinstance(workspace, str):
        workspace = new_workspace(_lib.prefill_workspace_bytes(d), qkv.device)
    _lib.check(_lib.prefill_rope_ws_raw(d, rope_mode, rope_base, qkv.data_ptr(), k_cache.data_ptr(),
                                        v_cache.data_ptr(), out.data_ptr(), lse.data_ptr() if lse is not None else 0,
                                        workspace.data_ptr(), workspace.numel(), _stream()))
    return out, lse


def linear(x, weights, *, out=None, gamma=None, bias=None, eps=1e-5, accumulate=False, out_f16=False):
    """mx_linear: x f32 [M][>= K]; weights: one f16 [N][K] tensor or a list of them (same shape, one launch);
    out: matching output tensor(s) (f32, or f16 with out_f16), created if None; gamma f32 [K] turns on the RMS norm;
    bias: f32 [N] tensor or list (None entries allowed). Returns the output tensor or list."""
    r = _native().linear(x, weights, out, gamma, bias, eps, accumulate, out_f16)
    if r is not None:
        return _result(r)
    single = isinstance(weights, torch.Tensor)
    ws_list = [weights] if single else list(weights)
    _rows(x, "x", torch.float32)
    N, K = ws_list[0].shape
    for w in ws_list:
        _rows(w, "weight")
        if tuple(w.shape) != (N, K) or w.stride(0) != K:
            raise ValueError("weights must be contiguous [N][K] tensors of one shape")
    odt = torch.float16 if out_f16 else torch.float32
    if out is None:
        outs = [torch.empty(x.shape[0], N, dtype=odt, device=x.device) for _ in ws_list]
    else:
        outs = [out] if single else list(out)
    for o in outs:
        _rows(o, "out", odt)
    if len({o.stride(0) for o in outs}) != 1:
        raise ValueError("outputs must share one row stride")
    bl = None
    if bias is not None:
        bl = [bias] if isinstance(bias, torch.Tensor) else list(bias)
    flags = ((_lib.LINEAR_RMS_NORM if gamma is not None else 0) | (_lib.LINEAR_ACCUMULATE if accumulate else 0) |
             (_lib.LINEAR_BIAS if bl is not None else 0) | (_lib.LINEAR_OUT_F16 if out_f16 else 0))
    d = _lib.MxLinearDesc(M=x.shape[0], N=N, K=K, flags=flags, x_stride=x.stride(0), y_stride=outs[0].stride(0),
                          eps=eps, reserved=0)
    need = _lib.linear_call_workspace_bytes(d, len(ws_list))
    ws = torch.empty(max(need, 256), dtype=torch.uint8, device=x.device) if need else None
    _lib.check(_lib.linear_raw(d, [w.data_ptr() for w in ws_list], x.data_ptr(), [o.data_ptr() for o in outs],
                               gamma.data_ptr() if gamma is not None else 0,
                               None if bl is None else [b.data_ptr() if b is not None else 0 for b in bl],
                               ws.data_ptr() if ws is not None else 0, ws.numel() if ws is not None else 0,
                               _stream()))
    return outs[0] if single else outs


_SA_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}


def self_attention(qkv, *, heads, scale=None, out=None, tuning=None):
    """mx_self_attention, the IR's SelfAttention op: qkv [B][N][3E] contiguous (f32, f16 or bf16) -> y [B][N][E] of the
    same dtype. scale defaults to head_dim^-0.5. The workspace (if the shape needs one) comes from torch's allocator."""
    if _tuning(tuning) is None:
        r = _native().self_attention(qkv, heads, scale, out)
        if r is not None:
            return _result(r)
    if not qkv.is_cuda:
        raise ValueError("qkv must be a device tensor")
    if qkv.dim() != 3 or not qkv.is_contiguous() or qkv.dtype not in _SA_DTYPES:
        raise ValueError("qkv must be a contiguous [B][N][3E] f32/f16/bf16 tensor")
    B, N, E3 = qkv.shape
    if E3 % 3:
        raise ValueError("the last dimension of qkv must be a multiple of 3")
    E = E3 // 3
    if scale is None:
        scale = (E // heads) ** -0.5 if heads >= 1 and E % heads == 0 else 1.0
    d = _lib.MxSelfAttnDesc(batch=B, n_tok=N, heads=heads, embed=E, dtype=_SA_DTYPES[qkv.dtype], scale=scale)
    t = _lib.make_tuning(_tuning(tuning))
    if t is not None:
        d.tuning = _lib.ctypes.pointer(t)
    if out is None:
        out = torch.empty(B, N, E, dtype=qkv.dtype, device=qkv.device)
    nbytes = _lib.self_attention_workspace_bytes(d)  # 0 also for an invalid descriptor, which the call reports
    ws = torch.empty(nbytes, dtype=torch.uint8, device=qkv.device) if nbytes else None
    _lib.check(_lib.self_attention_raw(d, qkv.data_ptr(), out.data_ptr(), ws.data_ptr() if ws is not None else 0,
                                       nbytes, _stream()))
    return out


# ---- the paged cache ----

_PAGED_COUNTERS = 512 << 10  # bytes of counters at the start of a workspace
_PAGE_DTYPES = {torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}


def _paged_scales(scales, k_pages):
    """The checked scales of pages in 8 bits, or None for pages in 16."""
    if k_pages.dtype != torch.float8_e4m3fn:
        if scales is not None:
            raise ValueError("scales belong to float8_e4m3fn pages")
        return None
    if scales is None or len(scales) != 2:
        raise ValueError("float8_e4m3fn pages need scales: those of the keys and those of the values")
    n_pages, page_size, n_head_kv, _ = k_pages.shape
    k, v = scales
    for t in (k, v):
        if t.device != k_pages.device or t.dtype != torch.float8_e8m0fnu or tuple(t.shape) != (n_pages, n_head_kv, page_size) or t.stride(2) != 1:
            raise ValueError("scales must be float8_e8m0fnu [pages][kv heads][page size] tensors with unit stride along the page on the "
                             "pages' device")
    if any(n > 1 and a != b for n, a, b in zip(k.shape, k.stride(), v.stride())):
        raise ValueError("the scales of the keys and of the values must share their strides")
    return _lib.MxPagedScales(k=k.data_ptr(), v=v.data_ptr(), page_stride=k.stride(0), head_stride=k.stride(1))


def _paged_desc(rows, k_pages, v_pages, page_table, kv_len, cu_q, n_head, max_q=None, max_kv_len=None, dtype=None):
    """The checked cache of a paged call as a descriptor (its rows' and outputs' types and strides are the caller's). Every
    tensor has to be on the device of `rows`. dtype: the queries' type, where the pages have 8 bits."""
    for t, name in ((rows, "rows"), (k_pages, "k_pages"), (v_pages, "v_pages"), (page_table, "page_table"), (kv_len, "kv_len"),
                    (cu_q, "cu_q")):
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError(f"{name} must be a device tensor")
        if t.device != rows.device:
            raise ValueError(f"{name} is on {t.device}, the rows on {rows.device}")
    if k_pages.dim() != 4 or k_pages.stride(3) != 1 or (k_pages.dtype not in _PAGE_DTYPES and k_pages.dtype != torch.float8_e4m3fn):
        raise ValueError("k_pages must be a float16, bfloat16 or float8_e4m3fn [pages][page size][kv heads][head dim] tensor with unit "
                         "stride along the head dim")
    if v_pages.shape != k_pages.shape or v_pages.dtype != k_pages.dtype or any(
            n > 1 and a != b for n, a, b in zip(k_pages.shape, k_pages.stride(), v_pages.stride())):  # a lone page or head has no stride
        raise ValueError("v_pages must have the shape, strides and type of k_pages")
    if page_table.dim() != 2 or page_table.dtype != torch.int32 or (page_table.stride(1) != 1 and page_table.shape[1] > 1):
        raise ValueError("page_table must be an int32 [sequences][pages] tensor with unit stride along the pages")
    n_seq = page_table.shape[0]
    if n_seq > 1 and page_table.stride(0) < page_table.shape[1]:
        raise ValueError("the rows of page_table overlap")
    if kv_len.dtype != torch.int32 or kv_len.shape != (n_seq,) or not kv_len.is_contiguous():
        raise ValueError("kv_len must be a contiguous int32 tensor with an entry per sequence")
    if cu_q is not None and (cu_q.dtype != torch.int32 or cu_q.shape != (n_seq + 1,) or not cu_q.is_contiguous()):
        raise ValueError("cu_q must be a contiguous int32 tensor of one entry more than sequences")
    n_pages, page_size, n_head_kv, head_dim = k_pages.shape
    return _lib.MxPagedDesc(n_head=n_head, n_head_kv=n_head_kv, head_dim=head_dim, dtype=_PAGE_DTYPES[dtype or k_pages.dtype], n_seq=n_seq,
                            n_rows=rows.shape[0], page_size=page_size, n_pages=n_pages, max_pages=page_table.shape[1],
                            max_q=max_q or 0, max_kv_len=max_kv_len or 0, page_stride=k_pages.stride(0),
                            kv_stride=k_pages.stride(1), head_stride=k_pages.stride(2),
                            table_stride=max(page_table.stride(0), page_table.shape[1]), row_stride=rows.stride(0))


def paged_store(qkv, k_pages, v_pages, page_table, kv_len, *, n_head, rope_mode, rope_base=10000.0, cu_q=None, positions=None,
                axis_pairs=None, axis_restart=False, q=None, want_q=True, scales=None, q_dtype=None):
    """mx_paged_store, the append of a step's new tokens: qkv (f32, f16 or bf16) [rows][>= (n_head + 2 n_head_kv) hd] unrotated
    rows, each sequence's new tokens as cu_q has them (None: equally many each); kv_len counts them already. Their rotated keys
    and their values go into k_pages / v_pages ([pages][page size][kv heads][hd], f16 or bf16, any strides but the last). Returns
    the rotated queries, [rows][n_head hd] of the pages' type (None without want_q). positions: int32 [axes][rows] or [rows]
    (None: the cache positions); axis_pairs: rotary pairs of each axis (None: one axis); axis_restart: each axis has a frequency
    ladder of its own. Pages in 8 bits (mx_paged_store_e4m3): float8_e4m3fn pages with scales, those of the keys and of the values,
    float8_e8m0fnu [pages][kv heads][page size]; the queries then have the type q_dtype, or that of q, or of qkv if it has 16 bits, or
    float16."""
    if scales is None:
        r = _native().paged_store(qkv, k_pages, v_pages, page_table, kv_len, n_head, rope_mode, rope_base, cu_q, positions, axis_pairs,
                                  axis_restart, q, want_q) if q_dtype is None else None
    else:
        r = _native().paged_store_e4m3(qkv, k_pages, v_pages, page_table, kv_len, n_head, rope_mode, rope_base, cu_q, positions,
                                       axis_pairs, axis_restart, q, want_q, scales, q_dtype)
    if r is not None:
        return _result(r)
    if qkv.dtype not in _SA_DTYPES:
        raise ValueError("qkv must be float32, float16 or bfloat16")
    _rows(qkv, "qkv", qkv.dtype)
    eight = k_pages.dtype == torch.float8_e4m3fn
    if q_dtype is None:
        q_dtype = k_pages.dtype if not eight else q.dtype if q is not None else qkv.dtype if qkv.dtype in _PAGE_DTYPES else torch.float16
    if q_dtype not in _PAGE_DTYPES if eight else q_dtype != k_pages.dtype:
        raise ValueError("the queries must have the pages' type, or be float16 or bfloat16 beside pages in 8 bits")
    d = _paged_desc(qkv, k_pages, v_pages, page_table, kv_len, cu_q, n_head, dtype=q_dtype)
    s = _paged_scales(scales, k_pages)
    d.row_dtype = _SA_DTYPES[qkv.dtype]
    if qkv.shape[1] < (n_head + 2 * d.n_head_kv) * d.head_dim:
        raise ValueError("qkv must be [rows][>= (n_head + 2 n_head_kv) head_dim]")
    rope = _lib.make_paged_rope(rope_mode, rope_base, (d.head_dim // 2,) if axis_pairs is None else axis_pairs, axis_restart)
    if positions is not None:
        if positions.device != qkv.device or positions.dtype != torch.int32 or not positions.is_contiguous():
            raise ValueError("positions must be a contiguous int32 tensor on the rows' device")
        if tuple(positions.shape) != (rope.n_axes, d.n_rows) and not (rope.n_axes == 1 and tuple(positions.shape) == (d.n_rows,)):
            raise ValueError("positions must be [axes][rows]")
    if want_q and q is None:
        q = torch.empty(d.n_rows, n_head * d.head_dim, dtype=q_dtype, device=qkv.device)
    if q is not None:
        _out_rows(q, "q", q_dtype, d, qkv)
        d.out_stride = q.stride(0)
    with torch.cuda.device(qkv.device):
        _lib.check(_lib.paged_store_raw(d, rope, qkv.data_ptr(), _ptr(positions), k_pages.data_ptr(), v_pages.data_ptr(),
                                        page_table.data_ptr(), kv_len.data_ptr(), _ptr(cu_q), _ptr(q), _stream(), s))
    return q


def _ptr(t) -> int:
    return t.data_ptr() if t is not None else 0


def _out_rows(out, name, dtype, d, like):
    _rows(out, name, dtype)
    if out.device != like.device or out.shape[0] < d.n_rows or out.shape[1] < d.n_head * d.head_dim:
        raise ValueError(f"{name} must be [rows][>= n_head * head_dim] on the rows' device")


def _paged_attend(q, k_pages, v_pages, page_table, kv_len, cu_q, n_head, causal, scale, out, out_dtype, lse, want_lse, max_q,
                  max_kv_len, scales, workspace, call, nbytes):
    if k_pages.dtype == torch.float8_e4m3fn and q.dtype not in _PAGE_DTYPES:
        raise ValueError("q must be float16 or bfloat16 beside pages in 8 bits")
    _rows(q, "q", q.dtype if k_pages.dtype == torch.float8_e4m3fn else k_pages.dtype)
    d = _paged_desc(q, k_pages, v_pages, page_table, kv_len, cu_q, n_head, max_q, max_kv_len, q.dtype)
    s = _paged_scales(scales, k_pages)
    if q.shape[1] < n_head * d.head_dim:
        raise ValueError("q must be [rows][>= n_head * head_dim]")
    if out_dtype is None:
        out_dtype = q.dtype if out is None else out.dtype
    if out_dtype not in (q.dtype, torch.float32):
        raise ValueError(f"the output must be {q.dtype} or float32")
    if out is None:
        out = torch.empty(d.n_rows, n_head * d.head_dim, dtype=out_dtype, device=q.device)
    _out_rows(out, "out", out_dtype, d, q)
    if want_lse and lse is None:
        lse = torch.empty(d.n_rows, n_head, dtype=torch.float32, device=q.device)
    if lse is not None and (lse.dtype != torch.float32 or not lse.is_contiguous() or tuple(lse.shape) != (d.n_rows, n_head) or
                            lse.device != q.device):
        raise ValueError("lse must be a contiguous float32 [rows][n_head] tensor on the rows' device")
    d.row_dtype = _SA_DTYPES[out_dtype]
    d.causal = 1 if causal else 0
    d.scale = 1.0 / math.sqrt(d.head_dim) if scale is None else scale
    d.out_stride = out.stride(0)
    with torch.cuda.device(q.device):
        if workspace is None:
            need = nbytes(d)  # 0 also for an invalid descriptor, which the call reports
            workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
            if need:  # the counters at its start have to be zero, the partials behind them need not be
                _lib.check(_lib.decode_workspace_init(workspace.data_ptr(), min(need, _PAGED_COUNTERS), _stream()))
        elif workspace.device != q.device or not workspace.is_contiguous():
            raise ValueError("workspace must be a contiguous tensor on the rows' device")
        rest = (out.data_ptr(), _ptr(lse), workspace.data_ptr(), workspace.numel() * workspace.element_size(), _stream(), s)
        _lib.check(call(d, q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), page_table.data_ptr(), kv_len.data_ptr(),
                        *(() if cu_q is None else (cu_q.data_ptr(),)), *rest))
    return out, lse


def paged_decode(q, k_pages, v_pages, page_table, kv_len, *, n_head, n_q=1, causal=True, scale=None, out=None, out_dtype=None, lse=None,
                 want_lse=False, max_kv_len=None, scales=None, workspace=None):
    """mx_paged_decode: q [sequences * n_q][>= n_head hd], the n_q new rows of each sequence (rotated, of the pages' type), over
    its kv_len[b] keys in k_pages / v_pages; page_table int32 [sequences][pages] and kv_len int32 on the device. With causal, row
    t of the n_q sees the keys up to kv_len - n_q + t. max_kv_len: a length that no sequence is expected to pass, for the plan. The
    output has q's type or out_dtype=torch.float32; workspace: paged_decode_workspace_bytes from new_workspace, kept by
    the caller (None: made for this call). Pages in 8 bits (mx_paged_decode_e4m3): float8_e4m3fn with scales as paged_store's, q
    float16 or bfloat16. Returns (out, lse or None)."""
    if q.dim() == 2 and page_table.dim() == 2 and q.shape[0] != page_table.shape[0] * n_q:
        raise ValueError(f"q has {q.shape[0]} rows, not {n_q} for each of {page_table.shape[0]} sequences")
    if workspace is not None:
        args = (q, k_pages, v_pages, page_table, kv_len, None, n_head, causal, scale, out, out_dtype, lse, want_lse, None, max_kv_len,
                workspace)
        r = _native().paged_attend(*args) if scales is None else _native().paged_attend_e4m3(*args, scales)
        if r is not None:
            return _result(r)
    return _paged_attend(q, k_pages, v_pages, page_table, kv_len, None, n_head, causal, scale, out, out_dtype, lse, want_lse, None,
                         max_kv_len, scales, workspace, _lib.paged_decode_raw, _lib.paged_decode_workspace_bytes)


def paged_decode_shared(q, k_pages, v_pages, page_table, kv_len, cu_seq, prefix_len, *, n_head, n_q=1, causal=True, scale=None, out=None,
                        out_dtype=None, lse=None, want_lse=False, max_own_len=None, scales=None, workspace=None):
    """mx_paged_decode_shared: paged_decode of sequences that come in groups which share their first keys. cu_seq int32 [groups + 1]
    and prefix_len int32 [groups] on the device: sequences cu_seq[g] .. cu_seq[g + 1] - 1 have the first prefix_len[g] keys in common,
    in the pages that the group's first sequence has for them; kv_len counts them too, and every new row has to see them all. The
    shared keys are read once for a group. max_own_len: the most keys of a sequence behind its prefix (all, of one in no group), for the plan. workspace:
    paged_shared_workspace_bytes from new_workspace. Everything else as paged_decode. Returns (out, lse or None)."""
    if q.dim() == 2 and page_table.dim() == 2 and q.shape[0] != page_table.shape[0] * n_q:
        raise ValueError(f"q has {q.shape[0]} rows, not {n_q} for each of {page_table.shape[0]} sequences")
    if workspace is not None:
        r = _native().paged_attend_shared(q, k_pages, v_pages, page_table, kv_len, None, n_head, causal, scale, out, out_dtype, lse,
                                          want_lse, None, max_own_len, workspace, scales, cu_seq, prefix_len)
        if r is not None:
            return _result(r)
    for t, name in ((cu_seq, "cu_seq"), (prefix_len, "prefix_len")):
        if t.device != q.device or t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 tensor of one dimension on the rows' device")
    if cu_seq.shape[0] != prefix_len.shape[0] + 1:
        raise ValueError("cu_seq must have one entry more than prefix_len")
    prefix = _lib.MxPagedPrefix(n_groups=prefix_len.shape[0], cu_seq=cu_seq.data_ptr(), prefix_len=prefix_len.data_ptr())
    return _paged_attend(q, k_pages, v_pages, page_table, kv_len, None, n_head, causal, scale, out, out_dtype, lse, want_lse, None,
                         max_own_len, scales, workspace, lambda d, *rest: _lib.paged_decode_shared_raw(d, prefix, *rest),
                         lambda d: _lib.paged_decode_shared_workspace_bytes(d, prefix.n_groups))


def paged_prefill(q, k_pages, v_pages, page_table, kv_len, cu_q, *, n_head, causal=True, scale=None, out=None, out_dtype=None,
                  lse=None, want_lse=False, max_q=None, max_kv_len=None, scales=None, workspace=None):
    """mx_paged_prefill: packed prompts, rows cu_q[b] .. cu_q[b + 1] - 1 (cu_q int32 on the device) the last of sequence b's
    kv_len[b] keys, which the pages hold already. max_q: the most rows of a sequence, for the plan. workspace:
    paged_prefill_workspace_bytes from new_workspace, kept by the caller; an empty tensor: no workgroups share a tile. Everything
    else as paged_decode."""
    if cu_q is None:
        raise ValueError("cu_q must be given")
    if workspace is not None:
        args = (q, k_pages, v_pages, page_table, kv_len, cu_q, n_head, causal, scale, out, out_dtype, lse, want_lse, max_q, max_kv_len,
                workspace)
        r = _native().paged_attend(*args) if scales is None else _native().paged_attend_e4m3(*args, scales)
        if r is not None:
            return _result(r)
    return _paged_attend(q, k_pages, v_pages, page_table, kv_len, cu_q, n_head, causal, scale, out, out_dtype, lse, want_lse, max_q,
                         max_kv_len, scales, workspace, _lib.paged_prefill_raw, _lib.paged_prefill_workspace_bytes)


def paged_decode_workspace_bytes(*, n_head, n_head_kv, head_dim, n_q, n_seq, max_kv_len) -> int:
    """Bytes of a workspace for paged_decode of n_seq sequences of n_q rows and at most max_kv_len keys."""
    return _lib.paged_decode_workspace_bytes(_lib.MxPagedDesc(
        n_head=n_head, n_head_kv=n_head_kv, head_dim=head_dim, dtype=_lib.DTYPE_F16, n_seq=n_seq, n_rows=n_seq * n_q, max_kv_len=max_kv_len))


def paged_prefill_workspace_bytes(*, n_head, n_head_kv, head_dim, n_rows, n_seq, max_q, max_kv_len) -> int:
    """Bytes of a workspace for paged_prefill of n_rows rows of n_seq sequences, at most max_q rows and max_kv_len keys each."""
    return _lib.paged_prefill_workspace_bytes(_lib.MxPagedDesc(
        n_head=n_head, n_head_kv=n_head_kv, head_dim=head_dim, dtype=_lib.DTYPE_F16, n_seq=n_seq, n_rows=n_rows, max_q=max_q,
        max_kv_len=max_kv_len))


def paged_shared_workspace_bytes(*, n_head, n_head_kv, head_dim, n_q, n_seq, n_groups, max_own_len) -> int:
    """Bytes of a workspace for paged_decode_shared of n_seq sequences of n_q rows in n_groups groups, with at most max_own_len keys
    each behind the prefix."""
    return _lib.paged_decode_shared_workspace_bytes(_lib.MxPagedDesc(
        n_head=n_head, n_head_kv=n_head_kv, head_dim=head_dim, dtype=_lib.DTYPE_F16, n_seq=n_seq, n_rows=n_seq * n_q,
        max_kv_len=max_own_len), n_groups)
