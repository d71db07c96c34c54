"""ctypes binding of include/vitk.h (lib/libvitk.so).  Arguments may be torch CUDA tensors
(float32/int32, contiguous unless a pitch is passed separately), raw integer addresses or None."""
import ctypes as C
import os

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "lib", "libvitk.so")

ACT_NONE, ACT_GELU_FWD, ACT_GELU_BWD = 0, 1, 2
DK_REFERENCE, DK_EXACT = 0, 1
PATCH_REFERENCE, PATCH_IM2COL = 0, 1


class VitkError(RuntimeError):
    pass


class GemmArgs(C.Structure):
    _fields_ = [
        ("trans_a", C.c_int32), ("trans_b", C.c_int32),
        ("M", C.c_int32), ("N", C.c_int32), ("K", C.c_int32),
        ("A", C.c_void_p), ("lda", C.c_int64),
        ("B", C.c_void_p), ("ldb", C.c_int64),
        ("C", C.c_void_p), ("ldc", C.c_int64),
        ("alpha", C.c_float), ("act", C.c_int32),
        ("bias", C.c_void_p), ("residual", C.c_void_p), ("ldr", C.c_int64),
        ("aux", C.c_void_p), ("ldaux", C.c_int64),
        ("batch_outer", C.c_int32), ("batch_inner", C.c_int32),
        ("stride_a_outer", C.c_int64), ("stride_a_inner", C.c_int64),
        ("stride_b_outer", C.c_int64), ("stride_b_inner", C.c_int64),
        ("stride_c_outer", C.c_int64), ("stride_c_inner", C.c_int64),
        ("split_k", C.c_int32), ("reserved", C.c_int32),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t), ("colsum_b", C.c_void_p),
    ]


class CrossSdpaArgs(C.Structure):
    _fields_ = [
        ("B", C.c_int32), ("H", C.c_int32), ("Hkv", C.c_int32), ("Nq", C.c_int32), ("Nk", C.c_int32), ("dh", C.c_int32),
        ("scale", C.c_float), ("reserved", C.c_int32),
        ("q", C.c_void_p), ("ld_q", C.c_int64), ("k", C.c_void_p), ("ld_k", C.c_int64),
        ("v", C.c_void_p), ("ld_v", C.c_int64), ("key_len", C.c_void_p),
        ("out", C.c_void_p), ("ld_out", C.c_int64), ("stats", C.c_void_p),
        ("dout", C.c_void_p), ("ld_dout", C.c_int64), ("dq", C.c_void_p), ("ld_dq", C.c_int64),
        ("dk", C.c_void_p), ("ld_dk", C.c_int64), ("dv", C.c_void_p), ("ld_dv", C.c_int64),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t),
    ]


class NewtonSchulzArgs(C.Structure):
    _fields_ = [
        ("rows", C.c_int32), ("cols", C.c_int32), ("batch", C.c_int32), ("steps", C.c_int32),
        ("x", C.c_void_p), ("ld_x", C.c_int64), ("stride_x", C.c_int64),
        ("out", C.c_void_p), ("ld_out", C.c_int64), ("stride_out", C.c_int64),
        ("a", C.c_float), ("b", C.c_float), ("c", C.c_float), ("eps", C.c_float),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t),
    ]


class MuonArgs(C.Structure):
    _fields_ = [
        ("rows", C.c_int32), ("cols", C.c_int32), ("batch", C.c_int32), ("steps", C.c_int32),
        ("p", C.c_void_p), ("g", C.c_void_p), ("m", C.c_void_p), ("ld", C.c_int64), ("stride", C.c_int64),
        ("lr", C.c_float), ("momentum", C.c_float), ("weight_decay", C.c_float), ("update_scale", C.c_float),
        ("grad_scale", C.c_float), ("nesterov", C.c_int32),
        ("a", C.c_float), ("b", C.c_float), ("c", C.c_float), ("eps", C.c_float),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t),
    ]


_p, _i32, _i64, _u64, _f, _sz = C.c_void_p, C.c_int32, C.c_int64, C.c_uint64, C.c_float, C.c_size_t

# name -> (restype, argtypes); every function of include/vitk.h
SIGNATURES = {
    "vitk_version": (C.c_int, []),
    "vitk_last_error": (C.c_char_p, []),
    "vitk_init": (C.c_int, [C.c_int]),
    "vitk_gemm_f32": (C.c_int, [C.POINTER(GemmArgs), _p]),
    "vitk_gemm_pair_f32": (C.c_int, [C.POINTER(GemmArgs), C.POINTER(GemmArgs), _p]),
    "vitk_gemm_workspace_bytes": (_sz, [C.POINTER(GemmArgs)]),
    "vitk_gemm_profile_enable": (C.c_int, [C.c_int]),
    "vitk_gemm_profile_read": (C.c_int, [C.c_int, C.POINTER(C.c_double), C.POINTER(C.c_double),
                                         C.POINTER(C.c_int64), C.c_int]),
    "vitk_gemm_variant_name": (C.c_char_p, [C.c_int]),
    "vitk_gemm_small_enable": (C.c_int, [C.c_int]),
    "vitk_set_planning_cu_count": (C.c_int, [C.c_int]),
    "vitk_sdpa_tile16_enable": (C.c_int, [C.c_int]),
    "vitk_sdpa_bwd_tile16_enable": (C.c_int, [C.c_int]),
    "vitk_colsum_workspace_bytes": (_sz, [_i64, _i64]),
    "vitk_colsum_f32": (C.c_int, [_p, _i64, _i64, _i64, _p, _p, _sz, _p]),
    "vitk_layernorm_bwd_workspace_bytes": (_sz, [_i64, _i64]),
    "vitk_layernorm_fwd": (C.c_int, [_p, _i64, _i64, _i64, _p, _p, _f, _p, _p, _p, _p]),
    "vitk_layernorm_bwd": (C.c_int, [_p, _p, _p, _p, _p, _i64, _i64, _i64, _p, _p, _p, _p, _p, _sz, _p]),
    "vitk_layernorm_bwd_static_max_d": (_sz, []),
    "vitk_layernorm_small_enable": (C.c_int, [C.c_int]),
    "vitk_layernorm_bwd_static": (C.c_int, [_p, _p, _p, _p, _p, _i64, _i64, _i64, _p, _p, _p, _p, _p]),
    "vitk_gelu_fwd": (C.c_int, [_p, _i64, _p, _p]),
    "vitk_gelu_bwd": (C.c_int, [_p, _p, _i64, _p, _p]),
    "vitk_dropout_fwd": (C.c_int, [_p, _i64, _f, _u64, _u64, _p, _p, _p]),
    "vitk_dropout_bwd": (C.c_int, [_p, _p, _i64, _p, _p]),
    "vitk_dropout_residual_fwd": (C.c_int, [_p, _p, _i64, _f, C.c_uint64, C.c_uint64, _p, _p, _p]),
    "vitk_dropout_stream_bwd": (C.c_int, [_p, _i64, _f, C.c_uint64, C.c_uint64, _p, _p]),
    "vitk_dropout_rows": (C.c_int, [_p, _p, _p, _i64, _i64, _i64, _f, C.c_uint64, C.c_uint64, _p, _p]),
    "vitk_add_f32": (C.c_int, [_p, _p, _i64, _p, _p]),
    "vitk_add3_f32": (C.c_int, [_p, _p, _p, _i64, _p, _p]),
    "vitk_scale_f32": (C.c_int, [_p, _f, _i64, _p, _p]),
    "vitk_fill_f32": (C.c_int, [_p, _f, _i64, _p]),
    "vitk_add_rowvec_f32": (C.c_int, [_p, _i64, _i64, _p, _p]),
    "vitk_copy2d_f32": (C.c_int, [_p, _i64, _p, _i64, _i64, _i64, _p]),
    "vitk_copy4d_f32": (C.c_int, [_p, C.POINTER(C.c_int64), C.POINTER(C.c_int64), _p, _p]),
    "vitk_softmax_rows": (C.c_int, [_p, _i64, _i64, _i64, _p, _p]),
    "vitk_softmax_rows_bwd": (C.c_int, [_p, _p, _i64, _i64, _i64, _f, _p, _p]),
    "vitk_dk_reference_scatter": (C.c_int, [_p, _i32, _i32, _i32, _i32, _p, _i64, _p]),
    "vitk_gather_rows_f32": (C.c_int, [_p, _i64, _p, _i64, _i64, _p, _p]),
    "vitk_augment_f32": (C.c_int, [_p, _i64, _p, _p, _i64, _i32, _i32, _i32, _p, _p]),
    "vitk_sdpa_head_kernels_enable": (C.c_int, [C.c_int]),
    "vitk_sdpa_supported": (C.c_int, [_i32, _i32]),
    "vitk_sdpa_fwd": (C.c_int, [_p, _p, _p, _i64, _i32, _i32, _i32, _i32, _f, _p, _i64, _p, _p]),
    "vitk_sdpa_bwd_workspace_bytes": (_sz, [_i32, _i32, _i32]),
    "vitk_sdpa_bwd": (C.c_int, [_p, _p, _p, _i64, _p, _p, _i64, _p, _i32, _i32, _i32, _i32, _f, _i32, _p, _p, _p, _i64,
                                _p, _sz, _p]),
    "vitk_sdpa_row_supported": (C.c_int, [_i32, _i32]),
    "vitk_sdpa_row_fwd": (C.c_int, [_p, _i64, _p, _p, _i64, _i32, _i32, _i32, _i32, _f, _p, _i64, _p, _p]),
    "vitk_sdpa_row_bwd": (C.c_int, [_p, _i64, _p, _p, _i64, _p, _p, _i64, _p, _i32, _i32, _i32, _i32, _f, _i32, _p, _i64,
                                    _p, _p, _i64, _p]),
    "vitk_cross_sdpa_fwd_workspace_bytes": (_sz, [C.POINTER(CrossSdpaArgs)]),
    "vitk_cross_sdpa_fwd": (C.c_int, [C.POINTER(CrossSdpaArgs), _p]),
    "vitk_cross_sdpa_bwd_workspace_bytes": (_sz, [C.POINTER(CrossSdpaArgs)]),
    "vitk_cross_sdpa_bwd": (C.c_int, [C.POINTER(CrossSdpaArgs), _p]),
    "vitk_embedding_fwd": (C.c_int, [_p, _i64, _p, _i64, _i64, _f, _p, _p]),
    "vitk_embedding_bwd_workspace_bytes": (_sz, [_i64, _i64, _i64]),
    "vitk_embedding_bwd": (C.c_int, [_p, _p, _i64, _i64, _i64, _f, _i32, _p, _p, _sz, _p]),
    "vitk_newton_schulz_workspace_bytes": (_sz, [_i32, _i32, _i32]),
    "vitk_newton_schulz_f32": (C.c_int, [C.POINTER(NewtonSchulzArgs), _p]),
    "vitk_muon_workspace_bytes": (_sz, [_i32, _i32, _i32]),
    "vitk_muon_f32": (C.c_int, [C.POINTER(MuonArgs), _p]),
    "vitk_add2d_f32": (C.c_int, [_p, _i64, _p, _i64, _i64, _i64, _p]),
    "vitk_patch_gather": (C.c_int, [_p, _i32, _i32, _i32, _i32, _i32, _p, _p]),
    "vitk_patch_scatter_bwd": (C.c_int, [_p, _i32, _i32, _i32, _i32, _i32, _p, _p]),
    "vitk_embed_assemble": (C.c_int, [_p, _p, _p, _i32, _i32, _i32, _p, _p]),
    "vitk_embed_split_bwd": (C.c_int, [_p, _i32, _i32, _i32, _p, _p]),
    "vitk_cls_gather": (C.c_int, [_p, _i32, _i32, _i32, _p, _p]),
    "vitk_cls_scatter": (C.c_int, [_p, _i32, _i32, _i32, _p, _p]),
    "vitk_softmax_ce": (C.c_int, [_p, _p, _i32, _i32, _p, _f, _p, _p, _p, _p, _sz, _p]),
    "vitk_argmax_rows": (C.c_int, [_p, _i32, _i32, _p, _p]),
    "vitk_adam_l2": (C.c_int, [_p, _p, _p, _p, _i64, _f, _f, _f, _f, _f, _f, _f, _f, _p]),
}

_dll = None


def dll():
    """The loaded library.  Raises (never falls back) when it has not been built."""
    global _dll
    if _dll is None:
        if not os.path.exists(LIB_PATH):
            raise VitkError(f"{LIB_PATH} is missing: build it with `make -C visiontransformer_amd` "
                            "(or __graft_entry__.build()); there is no CPU fallback")
        d = C.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(d, name)
            fn.restype, fn.argtypes = res, args
        _dll = d
    return _dll


def ptr(t):
    if t is None:
        return None
    if isinstance(t, int):
        return t
    return t.data_ptr()


_raw_stream = None


def stream(device=None):
    """Handle of torch's current stream on the current device, which has to be `device` if one is named.  (Building
    the Stream object for it takes 2.5 us, as much as the smallest kernels here, so the handle is asked for by itself
    where torch offers that: 0.3 us.)"""
    global _raw_stream
    import torch
    if _raw_stream is None:
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
            lambda device: torch.cuda.current_stream(device).cuda_stream)
    current = torch.cuda.current_device()
    if device is not None and device != current:
        raise VitkError(f"the tensors are on device {device}, the current one is {current}")
    return _raw_stream(current)


def _stream_for(args, st):
    """`st`, or the current stream; arguments made from tensors know their device."""
    current = stream(getattr(args, "device", None))
    return current if st is None else st


def _one_device(*tensors):
    devices = {t.get_device() for t in tensors if t is not None}
    if len(devices) != 1:
        raise VitkError(f"tensors on different devices: {sorted(devices)}")
    return devices.pop()


def check(rc):
    if rc != 0:
        raise VitkError(dll().vitk_last_error().decode())


def call(name, *args):
    """Call a status-returning entry point, converting tensors to addresses and raising on error."""
    fn = getattr(dll(), name)
    conv = [ptr(a) if (at is _p) else a for a, at in zip(args, fn.argtypes)]
    assert len(conv) == len(fn.argtypes), (name, len(conv), len(fn.argtypes))
    check(fn(*conv))


def init(device=0):
    check(dll().vitk_init(device))


def _gemm_args(A, B, Cout, M, N, K, *, trans_a=False, trans_b=False, lda=None, ldb=None, ldc=None, alpha=1.0,
               act=ACT_NONE, bias=None, residual=None, ldr=None, aux=None, ldaux=None, batch_outer=1, batch_inner=1,
               stride_a=(0, 0), stride_b=(0, 0), stride_c=(0, 0), split_k=1, colsum_b=None, tile=None):
    a = GemmArgs()
    a.reserved = {None: 0, "64x64": 1, "128x64": 2, "64x128": 3}[tile]
    a.trans_a, a.trans_b, a.M, a.N, a.K = int(trans_a), int(trans_b), M, N, K
    a.A, a.B, a.C = ptr(A), ptr(B), ptr(Cout)
    a.lda = lda if lda is not None else (M if trans_a else K)
    a.ldb = ldb if ldb is not None else (K if trans_b else N)
    a.ldc = ldc if ldc is not None else N
    a.alpha, a.act = alpha, act
    a.bias, a.residual, a.aux = ptr(bias), ptr(residual), ptr(aux)
    a.ldr = ldr if ldr is not None else N
    a.ldaux = ldaux if ldaux is not None else N
    a.batch_outer, a.batch_inner = batch_outer, batch_inner
    a.stride_a_outer, a.stride_a_inner = stride_a
    a.stride_b_outer, a.stride_b_inner = stride_b
    a.stride_c_outer, a.stride_c_inner = stride_c
    a.split_k = split_k
    a.colsum_b = ptr(colsum_b)
    return a


def _give_workspace(a, workspace):
    """Attach `workspace` (or, for tests, a fresh torch buffer) when these arguments need one."""
    need = dll().vitk_gemm_workspace_bytes(C.byref(a))
    keep = None
    if need:
        if workspace is None:
            import torch
            keep = workspace = torch.empty(need // 4, dtype=torch.float32, device="cuda")
        a.workspace, a.workspace_bytes = ptr(workspace), workspace.numel() * 4
    return keep


def gemm(A, B, Cout, M, N, K, *, workspace=None, st=None, **kw):
    """C = epilogue(alpha * op(A) op(B)); see include/vitk.h.  With split_k != 1 and no workspace given,
    one is allocated with torch (tests only; the host layer passes its own).  tile: None = the
    library's choice; "64x64", "128x64", "64x128" force that output tile (tests, measurements)."""
    a = _gemm_args(A, B, Cout, M, N, K, **kw)
    keep = _give_workspace(a, workspace)
    check(dll().vitk_gemm_f32(C.byref(a), st if st is not None else stream()))
    return keep


def gemm_pair(dx, dw, st=None):
    """vitk_gemm_pair_f32: dx and dw are dicts of gemm() arguments (A, B, Cout, M, N, K, ...) of the two
    products of a Dense backward."""
    ax, aw = _gemm_args(**dx), _gemm_args(**dw)
    keep = (_give_workspace(ax, None), _give_workspace(aw, None))
    check(dll().vitk_gemm_pair_f32(C.byref(ax), C.byref(aw), st if st is not None else stream()))
    return keep


def _need(cond, message):
    if not cond:
        raise VitkError(message)


_DTYPES = {}


def _is(t, dtype):
    if not _DTYPES:
        import torch
        _DTYPES.update(float32=torch.float32, int32=torch.int32)
    return t.dtype is _DTYPES[dtype] and t.is_cuda


def _f32(name, t, shape=None):
    _need(_is(t, "float32"), f"{name}: a float32 CUDA tensor is needed")
    _need(shape is None or tuple(t.shape) == tuple(shape), f"{name}: shape {tuple(t.shape)}, expected {shape}")


def _room(workspace):
    """Address and bytes of a workspace; a tensor with gaps or repeated elements (`expand`) has another extent."""
    if not (workspace.is_cuda and workspace.is_contiguous()):
        raise VitkError("workspace: a contiguous CUDA tensor is needed")
    return workspace.data_ptr(), workspace.nbytes


def _head_rows(name, t, shape):
    """Pitch of a [B, N, heads, dh] tensor whose rows (b, n) lie one after the other, heads packed."""
    _f32(name, t, shape)
    B, N, heads, dh = shape
    if t.numel() == 0:
        return heads * dh
    _need((dh == 1 or t.stride(3) == 1) and (heads == 1 or t.stride(2) == dh),
          f"{name}: the heads of a row have to be packed")
    if N > 1:
        ld = t.stride(1)
        _need(B == 1 or t.stride(0) == N * ld, f"{name}: batch entries have to follow each other at the row pitch")
    else:
        ld = t.stride(0) if B > 1 else heads * dh
    _need(ld >= heads * dh, f"{name}: rows overlap")
    return ld


def cross_sdpa_args(q, k, v, out, *, key_len=None, scale=None, stats=None, dout=None, dq=None, dk=None, dv=None,
                    workspace=None):
    """Arguments of cross_sdpa_fwd / cross_sdpa_bwd for q, out [B, Nq, H, dh] and k, v [B, Nk, Hkv, dh] (rows may be
    pitched, e.g. slices of a packed projection); the object keeps its tensors and, unless one is passed, a
    workspace.  Build it once and call as often as the same buffers are used.  Work that was put on another stream
    than torch's current one needs the object until it has ended, as any tensor there."""
    _need(q.dim() == 4 and k.dim() == 4, "cross_sdpa: q and k have four dimensions [B, N, heads, dh]")
    B, Nq, H, dh = q.shape
    Nk, Hkv = k.shape[1], k.shape[2]
    a = CrossSdpaArgs()
    a.B, a.H, a.Hkv, a.Nq, a.Nk, a.dh = B, H, Hkv, Nq, Nk, dh
    a.scale = dh ** -0.5 if scale is None else scale
    rows, keys = (B, Nq, H, dh), (B, Nk, Hkv, dh)
    for name, t, shape in (("q", q, rows), ("k", k, keys), ("v", v, keys), ("out", out, rows), ("dout", dout, rows),
                           ("dq", dq, rows), ("dk", dk, keys), ("dv", dv, keys)):
        if t is not None:
            setattr(a, name, ptr(t))
            setattr(a, "ld_" + name, _head_rows(name, t, shape))
    if key_len is not None:
        _need(_is(key_len, "int32") and key_len.is_contiguous()
              and tuple(key_len.shape) == (B,), "key_len: B contiguous int32 values on the GPU are needed")
        a.key_len = ptr(key_len)
    if stats is not None:
        _f32("stats", stats)
        _need(stats.is_contiguous() and stats.numel() == B * H * Nq * 2, "stats: [B*H, Nq, 2] contiguous is needed")
        a.stats = ptr(stats)
    need = dll().vitk_cross_sdpa_fwd_workspace_bytes(C.byref(a))
    if dq is not None:
        need = max(need, dll().vitk_cross_sdpa_bwd_workspace_bytes(C.byref(a)))
    if need and workspace is None:
        import torch
        workspace = torch.empty((need + 3) // 4, dtype=torch.float32, device=q.device)
    if workspace is not None:
        a.workspace, a.workspace_bytes = _room(workspace)
    a.keep = (q, k, v, out, key_len, stats, dout, dq, dk, dv, workspace)
    a.device = _one_device(*a.keep)
    return a


def cross_sdpa_fwd(args, st=None):
    """Softmax attention of args.q over args.k / args.v; see include/vitk.h."""
    check(dll().vitk_cross_sdpa_fwd(C.byref(args), _stream_for(args, st)))


def cross_sdpa_bwd(args, st=None):
    check(dll().vitk_cross_sdpa_bwd(C.byref(args), _stream_for(args, st)))


def _rows_2d(name, t, dtype="float32"):
    if not (_is(t, dtype) and t.is_contiguous()):
        raise VitkError(f"{name}: a contiguous {dtype} CUDA tensor is needed")


def embedding_fwd(table, index, out, *, scale=1.0, st=None):
    """out[i] = scale * table[index[i]]; an index outside the table gives zeros."""
    _rows_2d("table", table), _rows_2d("out", out), _rows_2d("index", index, "int32")
    V, D = table.shape
    rows = index.numel()
    _need(out.numel() == rows * D, f"out: {rows} rows of {D} are needed")
    current = stream(_one_device(table, index, out))
    check(dll().vitk_embedding_fwd(ptr(table), V, ptr(index), rows, D, scale, ptr(out), current if st is None else st))


def embedding_bwd(dout, index, dtable, *, scale=1.0, accumulate=False, workspace=None, st=None):
    """dtable[t] (+)= scale * sum of dout[i] over index[i] == t.  Without a workspace one is allocated."""
    _rows_2d("dout", dout), _rows_2d("dtable", dtable), _rows_2d("index", index, "int32")
    V, D = dtable.shape
    rows = index.numel()
    _need(dout.numel() == rows * D, f"dout: {rows} rows of {D} are needed")
    if workspace is None:
        import torch
        need = dll().vitk_embedding_bwd_workspace_bytes(rows, V, D)
        _need(need == 0 or st is None, "embedding_bwd: another stream than the current one needs a workspace of its own")
        workspace = torch.empty((need + 3) // 4, dtype=torch.float32, device=dout.device)
    room = _room(workspace)
    current = stream(_one_device(dout, index, dtable, workspace))
    check(dll().vitk_embedding_bwd(ptr(dout), ptr(index), rows, V, D, scale, int(bool(accumulate)), ptr(dtable), *room,
                                   current if st is None else st))
    return workspace


def _matrices(name, t, rows=None):
    """(batch, rows, cols, ld, stride) of a [batch, rows, cols] or [rows, cols] tensor with unit column stride."""
    _f32(name, t)
    _need(t.dim() in (2, 3), f"{name}: [rows, cols] or [batch, rows, cols] is needed")
    if t.dim() == 2:
        t = t.unsqueeze(0)
    batch, r, c = t.shape
    _need(c <= 1 or t.stride(2) == 1, f"{name}: unit column stride is needed")
    ld = t.stride(1) if r > 1 else max(c, 1)
    return batch, r, c, ld, t.stride(0) if batch > 1 else r * ld


def newton_schulz_args(x, out, *, steps=5, coefficients=(3.4445, -4.7750, 2.0315), eps=1e-7, workspace=None):
    """Arguments of newton_schulz for [batch, rows, cols] (or one matrix); see include/vitk.h."""
    a = NewtonSchulzArgs()
    a.batch, a.rows, a.cols, a.ld_x, a.stride_x = _matrices("x", x)
    shape = _matrices("out", out)
    _need(shape[:3] == (a.batch, a.rows, a.cols), "out: the shape of x is needed")
    a.ld_out, a.stride_out = shape[3:]
    a.x, a.out = ptr(x), ptr(out)
    a.steps, a.eps = steps, eps
    a.a, a.b, a.c = coefficients
    need = dll().vitk_newton_schulz_workspace_bytes(a.rows, a.cols, a.batch)
    return _with_workspace(a, need, workspace, x, (x, out))


def muon_args(p, g, m, *, lr, momentum=0.95, weight_decay=0.0, update_scale=1.0, grad_scale=1.0, nesterov=True, steps=5,
              coefficients=(3.4445, -4.7750, 2.0315), eps=1e-7, workspace=None):
    """Arguments of muon for parameters, gradients and momentum of one layout; see include/vitk.h."""
    a = MuonArgs()
    a.batch, a.rows, a.cols, a.ld, a.stride = _matrices("p", p)
    for name, t in (("g", g), ("m", m)):
        _need(_matrices(name, t) == (a.batch, a.rows, a.cols, a.ld, a.stride), f"{name}: the layout of p is needed")
    a.p, a.g, a.m = ptr(p), ptr(g), ptr(m)
    a.lr, a.momentum, a.weight_decay, a.update_scale, a.grad_scale = lr, momentum, weight_decay, update_scale, grad_scale
    a.nesterov, a.steps, a.eps = int(bool(nesterov)), steps, eps
    a.a, a.b, a.c = coefficients
    need = dll().vitk_muon_workspace_bytes(a.rows, a.cols, a.batch)
    return _with_workspace(a, need, workspace, p, (p, g, m))


def _with_workspace(a, need, workspace, like, keep):
    if need and workspace is None:
        import torch
        workspace = torch.empty((need + 3) // 4, dtype=torch.float32, device=like.device)
    if workspace is not None:
        a.workspace, a.workspace_bytes = _room(workspace)
    a.keep = keep + (workspace,)
    a.device = _one_device(*a.keep)
    return a


def newton_schulz(args, st=None):
    check(dll().vitk_newton_schulz_f32(C.byref(args), _stream_for(args, st)))


def muon(args, st=None):
    check(dll().vitk_muon_f32(C.byref(args), _stream_for(args, st)))


def planning_cu_count(cus):
    """Plans (kernel routes, split counts, tile shapes) as on a device with `cus` CUs; 0 = this device's."""
    check(dll().vitk_set_planning_cu_count(int(cus)))


def gemm_small(enable):
    """Route small problems to the one-wave-per-tile kernel (the default) or keep them on the tiled one."""
    check(dll().vitk_gemm_small_enable(int(enable)))


def sdpa_tile16(enable):
    """Attention (forward and backward) of head dimensions 33..64 on 16-row tiles (the default) or on the 32-row kernels."""
    check(dll().vitk_sdpa_tile16_enable(int(bool(enable))))
    check(dll().vitk_sdpa_bwd_tile16_enable(int(enable)))  # (n >= 2: n heads per workgroup, for tests)


def gemm_profile(enable):
    check(dll().vitk_gemm_profile_enable(int(enable)))


def gemm_profile_read(reset=True):
    """Per kernel variant: dict(name, ms, flops, launches) for variants that were launched."""
    out = []
    for v in range(53):
        ms, fl, n = C.c_double(), C.c_double(), C.c_int64()
        check(dll().vitk_gemm_profile_read(v, C.byref(ms), C.byref(fl), C.byref(n), 0))
        if n.value:
            out.append(dict(name=dll().vitk_gemm_variant_name(v).decode(), ms=ms.value, flops=fl.value,
                            launches=n.value))
    if reset:
        check(dll().vitk_gemm_profile_read(0, None, None, None, 1))
    return out
