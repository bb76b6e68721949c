"""Per-kernel wrappers over the kernel-level C ABI (include/llmgpu_ops.h).

Arguments are torch CUDA tensors (used only as device allocations); every call
checks the status code and the device error word and raises on failure.
"""
import ctypes
import functools
import struct

import torch

from ._lib import load

EPI_BF16, EPI_F32, EPI_RESID, EPI_GELU, EPI_DGELU = 0, 1, 2, 3, 4


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _stream():
    return torch.cuda.current_stream().cuda_stream


class KernelError(RuntimeError):
    pass


def _check(rc, what):
    if rc != 0:
        raise KernelError(f"{what} failed with status {rc}")


def gemm(A, B, M, N, K, *, a_mn=False, b_mn=False, lda=None, ldb=None, epi=EPI_F32, out=None,
         ldo=None, accumulate=False, resid=None, ldr=None, aux=None, ld_aux=None, splits=1,
         col_group=0, group_stride=0, bn=0, err=None):
    """D[M,N] = A[M,K] @ B[N,K]^T on the tcgen05 GEMM kernel (bf16 in, fp32 acc)."""
    lib = load()
    dev = A.device
    if lda is None:
        lda = A.shape[-1]
    if ldb is None:
        ldb = B.shape[-1]
    if out is None:
        dt = torch.float32 if epi in (EPI_F32, EPI_RESID) else torch.bfloat16
        out = torch.zeros(M, N, dtype=dt, device=dev)
    if ldo is None:
        ldo = out.shape[-1]
    own_err = err is None
    if own_err:
        err = torch.zeros(1, dtype=torch.int32, device=dev)
    ws = None
    if splits > 1:
        ws = torch.empty(splits * M * N, dtype=torch.float32, device=dev)
    rc = lib.llmgpu_op_gemm(_ptr(A), lda, int(a_mn), _ptr(B), ldb, int(b_mn), M, N, K, epi,
                            _ptr(out), ldo, int(accumulate), _ptr(resid), ldr or 0, _ptr(aux),
                            ld_aux or 0, splits, _ptr(ws), col_group, group_stride, bn,
                            _ptr(err), _stream())
    _check(rc, "llmgpu_op_gemm")
    if own_err:
        torch.cuda.synchronize()
        if int(err.item()) != 0:
            raise KernelError(f"gemm device error code {int(err.item())}")
    return out


def _sync_check(rc, what):
    _check(rc, what)
    torch.cuda.synchronize()


def embed(tokens, wte, wpe, B, T):
    lib = load()
    C, V = wte.shape[1], wte.shape[0]
    x = torch.empty(B * T, C, dtype=torch.float32, device=wte.device)
    _sync_check(lib.llmgpu_op_embed(_ptr(tokens), _ptr(wte), _ptr(wpe), _ptr(x), B, T, C, V,
                                    _stream()), "embed")
    return x


def embed_bwd(tokens, dx, wte_grad, wpe_grad, B, T, accumulate_wpe=False):
    """wte_grad[tok mod V] += dx rows; wpe_grad (+)= the batch sum of dx rows (in place)."""
    lib = load()
    V, C = wte_grad.shape
    work = torch.empty(int(lib.llmgpu_op_embed_bwd_work(B, T, C)), dtype=torch.uint8,
                       device=dx.device)
    _sync_check(lib.llmgpu_op_embed_bwd(_ptr(tokens), _ptr(dx), _ptr(wte_grad), _ptr(wpe_grad),
                                        B, T, C, V, int(accumulate_wpe), _ptr(work), _stream()),
                "embed_bwd")


def norm_fwd(x, gamma, beta, rms=False):
    lib = load()
    rows, C = x.shape
    y = torch.empty(rows, C, dtype=torch.bfloat16, device=x.device)
    mean = torch.empty(rows, device=x.device)
    rstd = torch.empty(rows, device=x.device)
    _sync_check(lib.llmgpu_op_norm_fwd(_ptr(x), _ptr(gamma), _ptr(beta), _ptr(y), _ptr(mean),
                                       _ptr(rstd), rows, C, int(rms), _stream()), "norm_fwd")
    return y, mean, rstd


def norm_bwd(dy, x, gamma, mean, rstd, resid=None, rms=False, out=None):
    """dx = resid + the norm's input gradient; `out` (may be `resid` itself) receives dx."""
    lib = load()
    rows, C = x.shape
    dx = torch.empty_like(x) if out is None else out
    dx16 = torch.empty(rows, C, dtype=torch.bfloat16, device=x.device)
    dg, db, ds = (torch.empty(C, device=x.device) for _ in range(3))
    work = torch.empty(int(lib.llmgpu_op_norm_bwd_work(rows, C)), device=x.device)
    _sync_check(lib.llmgpu_op_norm_bwd(_ptr(dy), _ptr(x), _ptr(gamma), _ptr(mean), _ptr(rstd),
                                       _ptr(resid), _ptr(dx), _ptr(dx16), _ptr(dg), _ptr(db),
                                       _ptr(ds), _ptr(work), rows, C, int(rms), _stream()),
                "norm_bwd")
    return dx, dx16, dg, db, ds


def cross_entropy(logits16, V, tokens, scale, smoothing=0.0):
    lib = load()
    rows, Vp = logits16.shape
    loss = torch.empty(rows, device=logits16.device)
    _sync_check(lib.llmgpu_op_cross_entropy(_ptr(logits16), rows, V, Vp, _ptr(tokens),
                                            _ptr(loss), scale, smoothing, _stream()),
                "cross_entropy")
    return loss


def rope_table(T, hd, theta, device):
    """(cos, sin) of pos * theta^(-2j/hd), shape [T, hd/2, 2] fp32."""
    j = torch.arange(hd // 2, dtype=torch.float64)
    ang = torch.arange(T, dtype=torch.float64)[:, None] * theta ** (-2.0 * j / hd)[None, :]
    return torch.stack([ang.cos(), ang.sin()], -1).float().to(device).contiguous()


def attention_fwd(qkv, B, T, H, hd, rope=None, workspace=True):
    """Causal attention forward; with `workspace`, a head_dim below 64 runs zero-padded on the
    tcgen05 kernel (llmgpu_op_attention_fwd_ws), else on the mma.sync kernel."""
    lib = load()
    C = H * hd
    out = torch.empty(B * T, C, dtype=torch.bfloat16, device=qkv.device)
    lse = torch.empty(B, H, T, device=qkv.device)
    if workspace:
        nbytes = int(lib.llmgpu_op_attention_bwd_work(B, T, H, hd))
        work = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=qkv.device)
        rc = lib.llmgpu_op_attention_fwd_ws(_ptr(qkv), _ptr(out), _ptr(lse), B, T, H, hd,
                                            _ptr(rope), _ptr(work) if nbytes else None,
                                            _stream())
    else:
        rc = lib.llmgpu_op_attention_fwd(_ptr(qkv), _ptr(out), _ptr(lse), B, T, H, hd,
                                         _ptr(rope), _stream())
    _sync_check(rc, "attention_fwd")
    return out, lse


def attention_bwd(qkv, out, dout, lse, B, T, H, hd, rope=None):
    lib = load()
    dqkv = torch.zeros_like(qkv)
    dvec = torch.empty(B, H, T, device=qkv.device)
    nbytes = int(lib.llmgpu_op_attention_bwd_work(B, T, H, hd))
    work = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=qkv.device)
    _sync_check(lib.llmgpu_op_attention_bwd(_ptr(qkv), _ptr(out), _ptr(dout), _ptr(lse),
                                            _ptr(dvec), _ptr(dqkv), B, T, H, hd, _ptr(rope),
                                            _ptr(work), _stream()), "attention_bwd")
    return dqkv


def swiglu_fwd(h13, F):
    lib = load()
    rows = h13.shape[0]
    g = torch.empty(rows, F, dtype=torch.bfloat16, device=h13.device)
    _sync_check(lib.llmgpu_op_swiglu_fwd(_ptr(h13), _ptr(g), rows, F, _stream()), "swiglu_fwd")
    return g


def swiglu_bwd(dg, h13, F):
    lib = load()
    rows = h13.shape[0]
    d = torch.empty_like(h13)
    _sync_check(lib.llmgpu_op_swiglu_bwd(_ptr(dg), _ptr(h13), _ptr(d), rows, F, _stream()),
                "swiglu_bwd")
    return d


GROUP_ROWS, GROUP_K = 1, 2


def gemm_grouped(A, B, M, N, K, grp, groups, mode, *, a_mn=False, b_mn=False, lda=None,
                 ldb=None, epi=EPI_F32, out=None, ldo=None, accumulate=False, aux=None,
                 ld_aux=None, b_grp_rows=0, out_grp_stride=0):
    """Grouped (per-expert) GEMM; `grp` is an int32 device tensor of groups+1 row offsets."""
    lib = load()
    if lda is None:
        lda = A.shape[-1]
    if ldb is None:
        ldb = B.shape[-1]
    if ldo is None:
        ldo = out.shape[-1]
    err = torch.zeros(1, dtype=torch.int32, device=A.device)
    rc = lib.llmgpu_op_gemm_grouped(_ptr(A), lda, int(a_mn), _ptr(B), ldb, int(b_mn), M, N, K,
                                    epi, _ptr(out), ldo, int(accumulate), _ptr(aux), ld_aux or 0,
                                    _ptr(grp), groups, mode, b_grp_rows, out_grp_stride,
                                    _ptr(err), _stream())
    _check(rc, "llmgpu_op_gemm_grouped")
    torch.cuda.synchronize()
    if int(err.item()) != 0:
        raise KernelError(f"grouped gemm device error code {int(err.item())}")
    return out


def moe_route(y, mean, rstd, gamma, beta, gate, B, T, k, rms=False):
    """Router: returns (probs [BT,E], idx [BT,k], wts [BT,k], ssum [BT])."""
    lib = load()
    C, E = gate.shape
    dev = y.device
    probs = torch.empty(B * T, E, dtype=torch.float32, device=dev)
    idx = torch.empty(B * T, k, dtype=torch.int32, device=dev)
    wts = torch.empty(B * T, k, dtype=torch.float32, device=dev)
    ssum = torch.empty(B * T, dtype=torch.float32, device=dev)
    _sync_check(lib.llmgpu_op_moe_route(_ptr(y), _ptr(mean), _ptr(rstd), _ptr(gamma), _ptr(beta),
                                        int(rms), _ptr(gate), B, T, C, E, k, _ptr(probs),
                                        _ptr(idx), _ptr(wts), _ptr(ssum), _stream()),
                "moe_route")
    return probs, idx, wts, ssum


def moe_dispatch(idx, B, T, E):
    """Dispatch: returns (grp [2E+1], row_of [BT,k], tok_of [BT*k + 128E])."""
    lib = load()
    k = idx.shape[1]
    dev = idx.device
    grp = torch.empty(2 * E + 1, dtype=torch.int32, device=dev)
    row_of = torch.empty(B * T, k, dtype=torch.int32, device=dev)
    tok_of = torch.empty(B * T * k + 128 * E, dtype=torch.int32, device=dev)
    _sync_check(lib.llmgpu_op_moe_dispatch(_ptr(idx), B, T, E, k, _ptr(grp), _ptr(row_of),
                                           _ptr(tok_of), _stream()), "moe_dispatch")
    return grp, row_of, tok_of


# ---- dropout, the linear layer and the loss head -------------------------------------------------
# These run asynchronously on the current stream of their tensors' device, like any torch operation,
# and allocate what they return (and their workspace) from torch's allocator, so they can be captured
# into a graph. Matrices are 2-D with neighbouring columns and any row stride; the matrices they
# return start their rows on 16 bytes (the row stride is rounded up to 8 elements), so that one
# operator's result can be another's operand. They are no autograd functions: what they return
# requires no gradient, whatever the operands do; the _bwd calls are the backward.
ACT = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}

_err_words = {}


def _err_word(device):
    """Address of the device's error word of these operators, in a capture too."""
    w = _err_words.get(device.index)
    if w is None:
        p = ctypes.c_void_p()
        with torch.cuda.device(device):
            rc = load().llmgpu_op_error_word(ctypes.byref(p))
        if rc != 0:
            raise KernelError(f"llmgpu_op_error_word failed with status {rc}")
        w = _err_words[device.index] = p.value
    return w


def check_device(device="cuda"):
    """Waits for the device and raises if a wait inside one of these operators' kernels gave up (its
    result, and those of the calls after it on any stream of the device, are then not to be used);
    the word is cleared. Nothing else reports it."""
    code = ctypes.c_int()
    with torch.cuda.device(torch.device(device)):
        rc = load().llmgpu_op_take_error(ctypes.byref(code))
    if rc != 0:
        raise KernelError(f"llmgpu_op_take_error failed with status {rc}")
    if code.value:
        raise KernelError(f"device error code {code.value}")


# llmgpu_op_call's number and block of each operator: integers and addresses in the order of the C
# call (the one unsigned word is `site`), the stream last, then the floats
_BLOCKS = {
    "llmgpu_op_dropout": (0, struct.Struct("11qQq1d").pack),
    "llmgpu_op_linear_fwd": (1, struct.Struct("8qQ13q1d").pack),
    "llmgpu_op_linear_bwd": (2, struct.Struct("12qQ14q1d").pack),
    "llmgpu_op_linear_ce_fwd": (3, struct.Struct("14q1d").pack),
    "llmgpu_op_linear_ce_bwd": (4, struct.Struct("22q2d").pack),
}
# the raw handle of a device's current stream, without making a Stream object (3 us a call)
_raw_stream = torch._C._cuda_getCurrentRawStream


def _call(name, device, ints, *floats):
    """The C entry point on the current stream of `device`, its arguments in one block."""
    op, pack = _BLOCKS[name]
    i = device.index
    fn = load().llmgpu_op_call
    if i == torch.cuda.current_device():
        rc = fn(op, pack(*ints, _raw_stream(i), *floats))
    else:
        with torch.cuda.device(device):
            rc = fn(op, pack(*ints, _raw_stream(i), *floats))
    if rc != 0:
        raise KernelError(f"{name} failed with status {rc}")


def _device_of(t, name):
    """The device of a 2-D CUDA tensor."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dim() != 2:
        raise KernelError(f"{name}: a 2-D CUDA tensor is needed")
    return t.device


def _matrix(t, name, dtypes, rows, cols, device, operand=False):
    """Checks a 2-D matrix argument and returns its address and row stride in elements."""
    if not isinstance(t, torch.Tensor) or t.get_device() != device.index:
        raise KernelError(f"{name}: a tensor on {device} is needed, as the first argument")
    if t.dtype not in dtypes:
        raise KernelError(f"{name}: {t.dtype} is not one of {[str(d) for d in dtypes]}")
    if t.shape != (rows, cols):
        raise KernelError(f"{name}: shape {tuple(t.shape)}, not {(rows, cols)}")
    ld, sc = t.stride()
    if sc != 1 and cols > 1:
        raise KernelError(f"{name}: neighbouring columns are needed")
    if rows <= 1:
        ld = (cols + 7) // 8 * 8
    elif ld < cols:
        raise KernelError(f"{name}: rows overlap (stride {ld} of {cols} columns)")
    p = t.data_ptr()
    if operand and (p % 16 or ld % 8) and rows and cols:
        raise KernelError(f"{name}: rows have to start on 16 bytes (address {p:#x}, stride {ld})")
    return p, ld


def _vector(t, name, dtype, n, device):
    """Checks a contiguous vector and returns its address."""
    if not isinstance(t, torch.Tensor) or t.get_device() != device.index or t.dtype != dtype or \
            t.shape != (n,) or not t.is_contiguous():
        raise KernelError(f"{name}: a contiguous {dtype} tensor of {n} on {device} is needed")
    return t.data_ptr()


def _new(rows, cols, dtype, device):
    """A new matrix whose rows start on 16 bytes, its address and row stride."""
    if dtype not in _FLOATS:
        raise KernelError(f"{dtype} is not one of {[str(d) for d in _FLOATS]}")
    ld = (cols + 7) // 8 * 8
    t = torch.empty_strided((rows, cols), (ld, 1), dtype=dtype, device=device)
    return t, t.data_ptr(), ld


@functools.lru_cache(maxsize=4096)
def _work_bytes(name, *sizes):
    """A workspace's size, which goes by the call's sizes alone."""
    return getattr(load(), name)(*sizes)


def _work(name, device, *sizes):
    """(tensor, address) of a new workspace, (None, 0) where none is needed."""
    n = _work_bytes(name, *sizes)
    if not n:
        return None, 0
    t = torch.empty(n, dtype=torch.uint8, device=device)
    return t, t.data_ptr()


def _drop(p, rng, device):
    if not 0.0 <= p <= 1.0:
        raise KernelError(f"p = {p} is not in [0, 1]")
    if rng is not None:
        return _vector(rng, "rng", torch.int64, 2, device)
    if p > 0.0:
        raise KernelError("dropout needs rng, an int64 tensor (seed, offset) on the device")
    return 0


def _act(act):
    if act not in ACT:
        raise KernelError(f"act: {act!r} is not one of {sorted(ACT)}")
    return ACT[act]


def _grad_w(dw, w_mn, rows, cols, device, accumulate):
    """(dw, address, row stride): the given weight gradient, or a new one in the weight's layout."""
    if w_mn:
        rows, cols = cols, rows
    if dw is None:
        if accumulate:
            raise KernelError("accumulate: dw has to be given")
        return _new(rows, cols, torch.bfloat16, device)
    if accumulate and dw.dtype != torch.float32:
        raise KernelError("accumulate: dw has to be f32")
    return (dw, *_matrix(dw, "dw", _FLOATS, rows, cols, device))


_FLOATS = (torch.float32, torch.bfloat16)
_U64 = 2 ** 64 - 1
_BF16 = (torch.bfloat16,)


def dropout_fwd(x, p, rng, site=0, resid=None, out=None, out_dtype=None):
    """resid + (kept ? x / (1 - p) : 0) over a 2-D x (f32 or bf16), in `out_dtype` (x's if not
    given). `rng`: int64 device tensor (seed, offset); `site` tells the dropouts of a step apart.
    The mask depends on (seed, offset + site, row, column) alone and p counts in steps of
    1 / 65536; see llmgpu_op_dropout. Between steps or micro-batches the offset has to move on by
    more than the largest site, or masks come back; data-parallel ranks need seeds of their own.
    `out` may be x or resid."""
    dev = _device_of(x, "x")
    rows, cols = x.shape
    px, ldx = _matrix(x, "x", _FLOATS, rows, cols, dev)
    prng = _drop(p, rng, dev)
    if not prng:
        raise KernelError("dropout needs rng, an int64 tensor (seed, offset) on the device")
    if out is None:
        out, po, ldo = _new(rows, cols, out_dtype or x.dtype, dev)
    elif out_dtype is not None and out.dtype != out_dtype:
        raise KernelError(f"out: {out.dtype} is not {out_dtype}")
    else:
        po, ldo = _matrix(out, "out", _FLOATS, rows, cols, dev)
    pr = ldr = 0
    if resid is not None:
        pr, ldr = _matrix(resid, "resid", (out.dtype,), rows, cols, dev)
    _call("llmgpu_op_dropout", dev,
          (px, x.dtype == torch.float32, ldx, pr, ldr, po, out.dtype == torch.float32, ldo, rows, cols,
           prng, site & _U64), p)
    return out


def dropout_bwd(dy, p, rng, site=0, out=None, out_dtype=None):
    """The gradient by x of dropout_fwd with the same (p, rng, site); the residual's is dy itself."""
    return dropout_fwd(dy, p, rng, site, out=out, out_dtype=out_dtype)


def _linear_shapes(x, w, w_mn):
    """(device, M, K, N, address and row stride of x, of w)"""
    dev = _device_of(x, "x")
    _device_of(w, "w")
    M, K = x.shape
    wr, wc = w.shape
    N = wc if w_mn else wr
    if N <= 0 or K <= 0:
        raise KernelError(f"an empty product: x {tuple(x.shape)}, w {tuple(w.shape)}")
    px, ldx = _matrix(x, "x", _BF16, M, K, dev, True)
    pw, ldw = _matrix(w, "w", _BF16, K if w_mn else N, N if w_mn else K, dev, True)
    return dev, M, K, N, px, ldx, pw, ldw


def linear_fwd(x, w, bias=None, act="none", p=0.0, rng=None, site=0, resid=None, w_mn=False,
               out=None, out_dtype=torch.bfloat16, save_pre=False):
    """resid + drop(act(x w^T + bias)) in one product. x [M, K] and w [N, K] (or [K, N] with
    `w_mn`) are bf16 with rows on 16 bytes, bias [N] f32, act one of ACT, (p, rng, site) as in
    dropout_fwd, resid of the result's type. Returns (y, pre): pre = x w^T + bias in bf16 when
    `save_pre` (linear_bwd needs it unless act is "none"), else None."""
    dev, M, K, N, px, ldx, pw, ldw = _linear_shapes(x, w, w_mn)
    a = _act(act)
    prng = _drop(p, rng, dev)
    pb = pr = pp = ldr = ldp = 0
    if bias is not None:
        pb = _vector(bias, "bias", torch.float32, N, dev)
    if out is None:
        out, po, ldo = _new(M, N, out_dtype, dev)
    else:
        po, ldo = _matrix(out, "out", _FLOATS, M, N, dev)
    if resid is not None:
        pr, ldr = _matrix(resid, "resid", (out.dtype,), M, N, dev)
    pre = None
    if save_pre:
        pre, pp, ldp = _new(M, N, torch.bfloat16, dev)
    work, pws = _work("llmgpu_op_linear_fwd_work", dev, M, N, K)
    _call("llmgpu_op_linear_fwd", dev,
          (px, ldx, pw, ldw, w_mn, pb, a, prng, site & _U64, pr, ldr, pp, ldp, po,
           out.dtype == torch.float32, ldo, M, N, K, pws, _err_word(dev)), p)
    return out, pre


def linear_bwd(dy, x, w, pre=None, act="none", p=0.0, rng=None, site=0, w_mn=False,
               dx_dtype=torch.bfloat16, dw=None, dbias=None, accumulate=False, need_dx=True,
               need_dw=True, need_dbias=True):
    """Gradients (dx, dw, dbias) of linear_fwd for the gradient dy [M, N] (f32 or bf16) of its
    result, with the forward's x, w, pre, act and (p, rng, site); the residual's gradient is dy. dw
    has w's layout, bf16 unless given; `accumulate` adds into the given dw (f32) and dbias. What
    is not needed is None."""
    dev, M, K, N, px, ldx, pw, ldw = _linear_shapes(x, w, w_mn)
    a = _act(act)
    prng = _drop(p, rng, dev)
    pdy, lddy = _matrix(dy, "dy", _FLOATS, M, N, dev)
    pp = ldp = pdx = lddx = pdw = lddw = pb = 0
    if act != "none":
        if pre is None:
            raise KernelError(f"act {act!r}: the backward needs pre")
        pp, ldp = _matrix(pre, "pre", _BF16, M, N, dev)
    dx = None
    if need_dx:
        dx, pdx, lddx = _new(M, K, dx_dtype, dev)
    if need_dw:
        dw, pdw, lddw = _grad_w(dw, w_mn, N, K, dev, accumulate)
    else:
        dw = None
    if need_dbias:
        if dbias is None:
            if accumulate:
                raise KernelError("accumulate: dbias has to be given")
            dbias = torch.empty(N, dtype=torch.float32, device=dev)
        pb = _vector(dbias, "dbias", torch.float32, N, dev)
    else:
        dbias = None
    work, pws = _work("llmgpu_op_linear_bwd_work", dev, M, N, K)
    _call("llmgpu_op_linear_bwd", dev,
          (pdy, dy.dtype == torch.float32, lddy, px, ldx, pw, ldw, w_mn, pp, ldp, a, prng, site & _U64,
           pdx, dx_dtype == torch.float32, lddx, pdw, need_dw and dw.dtype == torch.float32, lddw, pb,
           accumulate, M, N, K, pws, _err_word(dev)), p)
    return dx, dw, dbias


def _head_args(x, w, targets, smoothing, w_mn):
    if not 0.0 <= smoothing < 1.0:
        raise KernelError(f"smoothing = {smoothing} is not in [0, 1)")
    shapes = _linear_shapes(x, w, w_mn)
    return shapes, _vector(targets, "targets", torch.int32, shapes[1], shapes[0])


def linear_cross_entropy_fwd(x, w, targets, smoothing=0.0, w_mn=False):
    """Softmax cross-entropy of the logits x w^T without forming them in memory: (row_loss, lse),
    f32 [rows]. x [rows, C] and w [V, C] (or [C, V] with `w_mn`) are bf16 with rows on 16 bytes,
    targets int32 [rows]; a target outside [0, V) leaves its row out (loss 0). `smoothing` s:
    targets of 1 - s and s / (V - 1) elsewhere, in the loss as in the gradient."""
    (dev, rows, C, V, px, ldx, pw, ldw), pt = _head_args(x, w, targets, smoothing, w_mn)
    loss = torch.empty(rows, dtype=torch.float32, device=dev)
    lse = torch.empty(rows, dtype=torch.float32, device=dev)
    work, pws = _work("llmgpu_op_linear_ce_fwd_work", dev, rows, V)
    _call("llmgpu_op_linear_ce_fwd", dev,
          (px, ldx, pw, ldw, w_mn, pt, rows, C, V, loss.data_ptr(), lse.data_ptr(), pws,
           _err_word(dev)), smoothing)
    return loss, lse


def linear_cross_entropy_bwd(x, w, targets, lse, dloss=None, scale=1.0, smoothing=0.0, w_mn=False,
                             dx_dtype=torch.bfloat16, dw=None, accumulate=False, piece=0,
                             need_dx=True, need_dw=True):
    """Gradients (dx, dw) of sum(scale * dloss * row_loss) (dloss f32 [rows], ones if None), with
    the forward's arguments and its lse. The logits are formed again in pieces of `piece` columns of
    the vocabulary (a multiple of 256; 0: chosen by the library), which bounds the workspace. dw
    has w's layout, bf16 unless given; `accumulate` adds into the given f32 dw."""
    (dev, rows, C, V, px, ldx, pw, ldw), pt = _head_args(x, w, targets, smoothing, w_mn)
    if piece < 0 or piece % 256:
        raise KernelError(f"piece = {piece} is not a multiple of 256")
    pl = _vector(lse, "lse", torch.float32, rows, dev)
    pd = pdx = lddx = pdw = lddw = 0
    if dloss is not None:
        pd = _vector(dloss, "dloss", torch.float32, rows, dev)
    dx = None
    if need_dx:
        dx, pdx, lddx = _new(rows, C, dx_dtype, dev)
    if need_dw:
        dw, pdw, lddw = _grad_w(dw, w_mn, V, C, dev, accumulate)
    else:
        dw = None
    work, pws = _work("llmgpu_op_linear_ce_bwd_work", dev, rows, C, V, piece)
    _call("llmgpu_op_linear_ce_bwd", dev,
          (px, ldx, pw, ldw, w_mn, pt, pl, pd, rows, C, V, pdx, dx_dtype == torch.float32, lddx, pdw,
           need_dw and dw.dtype == torch.float32, lddw, accumulate, piece, pws, _err_word(dev)),
          scale, smoothing)
    return dx, dw
