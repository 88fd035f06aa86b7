"""Tensor-level wrappers over the C-ABI (include/eth_amd.h).

Each wrapper checks, on the host, that shapes, strides, dtypes and devices
match what the kernel and its launch grid assume, then enqueues the kernel on
the current stream.  There is no CPU fallback: CPU tensors raise.
"""

import ctypes
import functools
import itertools
import operator

import numpy as np

import torch

from . import _native as nat

_HALF_CODES = {torch.bfloat16: nat.ETH_BF16, torch.float16: nat.ETH_F16}


def _check_half(*ts):
    dt = ts[0].dtype
    code = _HALF_CODES.get(dt)
    if code is None:
        raise ValueError(f"expected bf16/fp16 tensors, got {dt}")
    for t in ts:
        if t.dtype != dt:
            raise ValueError(f"dtype mismatch {t.dtype} vs {dt}")
        if not t.is_cuda:
            raise ValueError("eth_amd kernels run on the GPU only (no CPU fallback)")
    return code


def _rows_cols(x):
    if not x.is_contiguous():
        raise ValueError("expected a contiguous tensor")
    cols = x.shape[-1]
    return x.numel() // cols if cols else 0, cols


# --------------------------------------------------------------------- GEMM --
def _matrix_layout(t):
    """(ld, kcontig-ready) of a 2-D view: returns (ld, row_major) where
    row_major means t[i, j] = base[i*ld + j]; column-major views (t.T of a
    row-major matrix) give row_major False."""
    if t.dim() != 2:
        raise ValueError("expected a 2-D operand")
    s0, s1 = t.stride()
    rows, cols = t.shape
    if s1 == 1 and s0 >= cols:
        return s0, True
    if s0 == 1 and s1 >= rows:
        return s1, False
    raise ValueError(f"operand with strides {t.stride()} is neither row- nor column-major")


_observer = None


def set_kernel_observer(fn):
    """fn(kind, phase, flops) is called right before ("begin") and after
    ("end") every GEMM ("gemm") and attention ("attn_fwd", "attn_bwd")
    launch, on the thread that launches it, with the launch's algorithmic
    FLOPs (the benchmark records HIP events on the launch stream with it);
    None disables it."""
    global _observer
    _observer = fn


def _observe(kind, phase, flops):
    obs = _observer
    if obs is not None:
        obs(kind, phase, flops)


def _splitk_splits(M, N, K, out):
    """Split-K factor for a product whose 256x256 tile grid is too small to
    fill the chip (at most 128 tiles): enough k-splits for about one
    workgroup per CU, each at least 1024 deep.  ([2048, 4096] x 16384 deep,
    128 tiles: 294 us in one pass, 208 us in two splits; three splits for up
    to 170 tiles, two rounds of a third, gained nothing.)"""
    tiles = -(-M // 256) * -(-N // 256)
    if tiles > 128 or N % 4 or out.stride(0) % 4 or out.data_ptr() % (4 * out.element_size()):
        return 1
    splits = 1
    while splits < 16 and tiles * splits * 2 <= 256 and K // (splits * 2) >= 1024:
        splits *= 2
    return splits


@functools.lru_cache(maxsize=4096)
def _splitk_pays(M, N, K, splits, a_kcontig, b_kcontig, out_code):
    """fp32 elements of workspace if the split-K form takes this product and
    finishes before the plain one, else 0 (by sizes, layout and type; the smaller
    tiles fill the chip without a second pass unless K is deep)."""
    if splits < 2 or K % 8 or 4 * (M + 256) * N >= 2**31:
        return 0
    if not nat.value("eth_gemm_splitk_pays", M, N, K, splits, a_kcontig, b_kcontig, out_code):
        return 0
    return nat.value("eth_gemm_splitk_workspace", M, N, splits) // 4


_side = {}
_side_launches = itertools.count(1)
_side_last = 0  # a value no earlier launch had, set at every side-stream launch


def side_stream(device):
    """The stream the weight-gradient GEMMs run on when overlapped with the
    data-gradient chain (default priority, one per device)."""
    st = _side.get(device)
    if st is None:
        st = torch.cuda.Stream(device=device)
        _side[device] = st
    return st


def mark_side_launch():
    """Note work about to be issued on a side stream."""
    global _side_last
    _side_last = next(_side_launches)


def side_mark():
    """Changes whenever side-stream work was issued (by any thread)."""
    return _side_last


def join_side_streams(since=None):
    """Make the current stream wait for all side-stream work (before main
    grads are read); with `since`, an earlier side_mark(), only if any was
    issued after it."""
    if since is not None and since == _side_last:
        return
    for dev, st in _side.items():
        torch.cuda.current_stream(dev).wait_stream(st)


def gemm(a, b, out=None, bias=None, accumulate=False, out_dtype=None, alpha=1.0):
    """out (+)= alpha * a @ b (+ bias), a: [M, K], b: [K, N] (any row/column-
    major 2-D views), out: [M, N] row-major.  fp32 `out` with accumulate=True
    adds into it."""
    code = _check_half(a, b)
    M, K = a.shape
    K2, N = b.shape
    if K != K2:
        raise ValueError(f"inner dimensions differ: {a.shape} @ {b.shape}")
    lda, a_row = _matrix_layout(a)
    ldb, b_row = _matrix_layout(b)
    # A(m,k) K-contiguous <=> a row-major; B(k,n) K-contiguous <=> b column-major
    a_kcontig = 1 if a_row else 0
    b_kcontig = 0 if b_row else 1
    if out is None:
        out = torch.empty(M, N, dtype=out_dtype or a.dtype, device=a.device)
    if out.dim() != 2 or out.shape != (M, N) or out.stride(1) != 1:
        raise ValueError("out must be a row-major [M, N] matrix")
    if accumulate and out.dtype != torch.float32:
        raise ValueError("accumulate needs an fp32 output")
    flags = 0
    if accumulate:
        flags |= nat.GEMM_ACCUMULATE
    if bias is not None:
        if bias.dtype != a.dtype or bias.numel() != N or not bias.is_contiguous():
            raise ValueError("bias must be a contiguous [N] tensor of the input dtype")
        flags |= nat.GEMM_BIAS
    _observe("gemm", "begin", 2.0 * M * N * K)
    splits = _splitk_splits(M, N, K, out)
    out_code = nat.dtype_code(out.dtype)
    partials = _splitk_pays(M, N, K, splits, a_kcontig, b_kcontig, out_code)
    if partials:
        # (a fresh buffer per call: two threads may share the stream)
        ws = torch.empty(partials, dtype=torch.float32, device=a.device)
        nat.call(
            "eth_gemm_splitk_out",
            nat.ptr(a), lda, a_kcontig,
            nat.ptr(b), ldb, b_kcontig,
            nat.ptr(out), out.stride(0), out_code,
            nat.ptr(bias), M, N, K, code, flags, float(alpha), splits, nat.ptr(ws),
            nat.stream_ptr(a.device),
        )
        _observe("gemm", "end", 2.0 * M * N * K)
        return out
    nat.call(
        "eth_gemm",
        nat.ptr(a), lda, a_kcontig,
        nat.ptr(b), ldb, b_kcontig,
        nat.ptr(out), out.stride(0), out_code,
        nat.ptr(bias), M, N, K, code, flags, float(alpha),
        nat.stream_ptr(a.device),
    )
    _observe("gemm", "end", 2.0 * M * N * K)
    return out


def linear(x2d, weight, bias=None):
    """F.linear: x2d [T, K] @ weight[N, K]^T (+ bias)."""
    return gemm(x2d, weight.t(), bias=bias)


# ---------------------------------------------------------------- LayerNorm --
def layer_norm_fwd(x, gamma, beta, eps=1e-5):
    code = _check_half(x, gamma, beta)
    rows, cols = _rows_cols(x)
    if gamma.numel() != cols or beta.numel() != cols:
        raise ValueError("gamma/beta must match the normalized size")
    y = torch.empty_like(x)
    mean = torch.empty(rows, dtype=torch.float32, device=x.device)
    rstd = torch.empty(rows, dtype=torch.float32, device=x.device)
    nat.call("eth_ln_fwd", nat.ptr(x), nat.ptr(gamma), nat.ptr(beta), nat.ptr(y), nat.ptr(mean), nat.ptr(rstd),
             rows, cols, float(eps), code, nat.stream_ptr(x.device))
    return y, mean, rstd


def layer_norm_fwd_sb(x, gamma, beta, eps=1e-5):
    """LayerNorm of a contiguous [s, b, h] x returned as [b, s, h] (the
    final LayerNorm after .transpose(0, 1).contiguous(), without the copy);
    mean / rstd in the output's row order."""
    code = _check_half(x, gamma, beta)
    if x.dim() != 3 or not x.is_contiguous():
        raise ValueError("x must be a contiguous [s, b, h] tensor")
    s, b, h = x.shape
    if gamma.numel() != h or beta.numel() != h:
        raise ValueError("gamma/beta must match the normalized size")
    y = torch.empty(b, s, h, dtype=x.dtype, device=x.device)
    mean = torch.empty(b * s, dtype=torch.float32, device=x.device)
    rstd = torch.empty(b * s, dtype=torch.float32, device=x.device)
    nat.call("eth_ln_fwd_sb", nat.ptr(x), nat.ptr(gamma), nat.ptr(beta), nat.ptr(y), nat.ptr(mean), nat.ptr(rstd),
             s, b, h, float(eps), code, nat.stream_ptr(x.device))
    return y, mean, rstd


def layer_norm_bwd_sb(dy, x, mean, rstd, gamma, dgamma, dbeta, accumulate):
    """Backward of layer_norm_fwd_sb: dy [b, s, h], x [s, b, h] -> dx [s, b, h];
    dgamma/dbeta fp32 stored or accumulated in place."""
    code = _check_half(dy, x, gamma)
    if x.dim() != 3 or not x.is_contiguous():
        raise ValueError("x must be a contiguous [s, b, h] tensor")
    s, b, h = x.shape
    if tuple(dy.shape) != (b, s, h) or not dy.is_contiguous():
        raise ValueError("dy must be a contiguous [b, s, h] tensor")
    for t in (dgamma, dbeta):
        if t.dtype != torch.float32 or t.numel() != h or not t.is_contiguous():
            raise ValueError("dgamma/dbeta must be contiguous fp32 [cols]")
    ws = torch.empty(nat.value("eth_ln_bwd_workspace", s * b, h), dtype=torch.float32, device=x.device)
    dx = torch.empty_like(x)
    nat.call("eth_ln_bwd_sb", nat.ptr(dy), nat.ptr(x), nat.ptr(mean), nat.ptr(rstd), nat.ptr(gamma), nat.ptr(dx),
             nat.ptr(dgamma), nat.ptr(dbeta), nat.ptr(ws), s, b, h, 1 if accumulate else 0, code,
             nat.stream_ptr(x.device))
    return dx


def layer_norm_bwd(dy, x, mean, rstd, gamma, dgamma, dbeta, accumulate, dresid=None, colsum=False):
    """dx (returned); dgamma/dbeta fp32 stored or accumulated in place.

    With `dresid` (the gradient of the residual branch that read the same x)
    the returned dx is bf16(bf16(dx_ln) + dresid).  With `colsum` as well,
    returns (dx, part): fp32 [groups, cols] column-sum partials of dx, folded
    by `reduce_partials` into a bias gradient."""
    code = _check_half(dy, x, gamma)
    rows, cols = _rows_cols(x)
    if dy.shape != x.shape or not dy.is_contiguous():
        raise ValueError("dy must match x")
    for t in (dgamma, dbeta):
        if t.dtype != torch.float32 or t.numel() != cols or not t.is_contiguous():
            raise ValueError("dgamma/dbeta must be contiguous fp32 [cols]")
    if dresid is not None:
        _check_half(dresid)
        if dresid.dtype != x.dtype or dresid.shape != x.shape or not dresid.is_contiguous():
            raise ValueError("dresid must be a contiguous tensor like x")
    elif colsum:
        raise ValueError("colsum needs dresid")
    ws = torch.empty(nat.value("eth_ln_bwd_workspace", rows, cols), dtype=torch.float32, device=x.device)
    part = None
    if colsum:
        part = torch.empty(nat.value("eth_ln_bwd_groups", rows, cols), cols, dtype=torch.float32, device=x.device)
    dx = torch.empty_like(x)
    nat.call("eth_ln_bwd_residual", nat.ptr(dy), nat.ptr(x), nat.ptr(mean), nat.ptr(rstd), nat.ptr(gamma),
             nat.ptr(dresid), nat.ptr(dx), nat.ptr(dgamma), nat.ptr(dbeta),
             nat.ptr(part), nat.ptr(ws), rows, cols, 1 if accumulate else 0, code,
             nat.stream_ptr(x.device))
    return (dx, part) if colsum else dx


def reduce_partials(part, out, accumulate):
    """out[c] (+)= sum_g part[g, c] (fp32), fixed summation order."""
    if part.dtype != torch.float32 or part.dim() != 2 or not part.is_contiguous():
        raise ValueError("part must be contiguous fp32 [groups, cols]")
    groups, cols = part.shape
    if out.dtype != torch.float32 or out.numel() != cols or not out.is_contiguous():
        raise ValueError("out must be contiguous fp32 [cols]")
    nat.call("eth_reduce_partials", nat.ptr(part), groups, cols, cols, nat.ptr(out), 1 if accumulate else 0,
             nat.stream_ptr(part.device))
    return out


def _norm_desc(x, post_gamma, post_beta, gate, residual_scale, gamma, beta, eps, rms):
    """(device index, descriptor) of residual norm operands: contiguous x
    [..., cols] and parameters [cols] of its type."""
    code = _HALF_CODES.get(x.dtype)
    if code is None:
        raise ValueError(f"expected bf16/fp16 tensors, got {x.dtype}")
    index = x.get_device()
    if index < 0:
        raise ValueError("eth_amd kernels run on the GPU only (no CPU fallback)")
    rows, cols = _rows_cols(x)
    if cols < 1 or cols % 8 or cols > 8192:
        raise ValueError(f"the normalized size must be a multiple of 8 up to 8192 (got {cols})")
    if rms and (post_beta is not None or beta is not None):
        raise ValueError("root-mean-square norms have no betas")
    if not rms and (post_beta is None or beta is None):
        raise ValueError("betas are needed (but for root-mean-square norms)")
    at, dtype, shape = [], x.dtype, (cols,)
    for name, t in (("post_gamma", post_gamma), ("post_beta", post_beta), ("gate", gate), ("gamma", gamma),
                    ("beta", beta)):
        if t is None:
            if name in ("post_gamma", "gamma"):
                raise ValueError(f"{name} is needed")
            at.append(None)
            continue
        place = t.data_ptr()
        if t.dtype != dtype or t.shape != shape or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous [{cols}] tensor of the input type")
        if place % 16:
            raise ValueError(f"{name} must be 16-byte aligned")
        if t.get_device() != index:
            _check_device(index, t)
        at.append(place)
    desc = nat.ResidualNormDesc(*at, rows, cols, float(residual_scale), float(eps), bool(rms), code)
    return index, desc


def _check_like(name, t, x):
    if t.shape != x.shape or t.dtype != x.dtype or not t.is_contiguous() or t.data_ptr() % 16:
        raise ValueError(f"{name} must be a contiguous, 16-byte aligned tensor like x")


def residual_norm_fwd(x, residual, post_gamma, post_beta, gate, residual_scale, gamma, beta, eps=1e-5, rms=False):
    """(h, y, stats): h = residual_scale * residual + gate * norm(x), y = norm(h)
    of h before its rounding, each norm with its gamma and beta; gate None: one.  With
    `rms` the norms are root-mean-square ones and have no betas (None).  stats
    [4, rows] fp32, for the backward."""
    index, desc = _norm_desc(x, post_gamma, post_beta, gate, residual_scale, gamma, beta, eps, rms)
    _check_device(index, residual)
    _check_like("x", x, x)
    _check_like("residual", residual, x)
    h, y = torch.empty_like(x), torch.empty_like(x)
    stats = torch.empty(4, desc.rows, dtype=torch.float32, device=x.device)
    _launch(index, "eth_residual_norm_fwd", ctypes.byref(desc), x.data_ptr(), residual.data_ptr(), h.data_ptr(),
            y.data_ptr(), stats.data_ptr())
    return h, y, stats


def residual_norm_bwd(x, residual, stats, dh, dy, post_gamma, post_beta, gate, residual_scale, gamma, beta, eps, rms, grads,
                      need_dx=True, need_dresidual=True):
    """(dx, dresidual) of residual_norm_fwd for the gradients dh of h and dy of y
    (one of them may be None), None where not needed.  `grads`: for post_gamma,
    post_beta, gate, gamma and beta a pair (tensor [cols] that the parameter's
    gradient is written to, whether it is added), or None; of the parameters'
    type, or fp32 (which alone can be added to); no two of them the same."""
    index, desc = _norm_desc(x, post_gamma, post_beta, gate, residual_scale, gamma, beta, eps, rms)
    given = [t for t in (dh, dy) if t is not None]
    if not given:
        raise ValueError("residual_norm_bwd needs dh or dy")
    _check_device(index, residual, stats, *given)
    for name, t in (("x", x), ("residual", residual), ("dh", dh), ("dy", dy)):
        if t is not None:
            _check_like(name, t, x)
    if stats.dtype != torch.float32 or stats.shape != (4, desc.rows) or not stats.is_contiguous():
        raise ValueError("stats must be the forward's fp32 [4, rows]")
    table = (nat.ResidualNormGrad * 5)()
    for i, (pair, param) in enumerate(zip(grads, (post_gamma, post_beta, gate, gamma, beta))):
        if pair is None:
            continue
        t, accumulate = pair
        fp32 = t.dtype == torch.float32
        if param is None or not fp32 and t.dtype != x.dtype or t.numel() != desc.cols or not t.is_contiguous():
            raise ValueError("a parameter's gradient must be a contiguous [cols] tensor of its type or fp32")
        if accumulate and not fp32:
            raise ValueError("accumulate needs an fp32 gradient")
        if t.get_device() != index:
            _check_device(index, t)
        table[i] = (t.data_ptr(), fp32, bool(accumulate))
    dx = torch.empty_like(x) if need_dx else None
    dresidual = torch.empty_like(x) if need_dresidual else None
    if not desc.rows:
        for pair in grads:
            if pair is not None and not pair[1]:
                pair[0].zero_()
        return dx, dresidual
    ws = torch.empty(nat.value("eth_residual_norm_workspace", desc.rows, desc.cols), dtype=torch.float32, device=x.device)
    _launch(index, "eth_residual_norm_bwd", ctypes.byref(desc), x.data_ptr(), residual.data_ptr(), stats.data_ptr(),
            nat.ptr(dh), nat.ptr(dy), nat.ptr(dx), nat.ptr(dresidual), table, ws.data_ptr())
    return dx, dresidual


# -------------------------------------------------------------- elementwise --
def bias_gelu_fwd(x, bias):
    code = _check_half(x, bias)
    rows, cols = _rows_cols(x)
    if bias.numel() != cols:
        raise ValueError("bias size mismatch")
    y = torch.empty_like(x)
    nat.call("eth_bias_gelu_fwd", nat.ptr(x), nat.ptr(bias), nat.ptr(y), rows, cols, code, nat.stream_ptr(x.device))
    return y


def bias_gelu_bwd(dy, x, bias, dbias=None, accumulate=False):
    """dx = dy * gelu_tanh'(x + b); with `dbias` (fp32 [cols]) the column
    sums of dx are stored or added into it in the same pass."""
    code = _check_half(dy, x, bias)
    rows, cols = _rows_cols(x)
    if dy.shape != x.shape or not dy.is_contiguous() or bias.numel() != cols:
        raise ValueError("shape mismatch")
    dx = torch.empty_like(x)
    if dbias is None:
        nat.call("eth_bias_gelu_bwd", nat.ptr(dy), nat.ptr(x), nat.ptr(bias), nat.ptr(dx), rows, cols, code,
                 nat.stream_ptr(x.device))
        return dx
    if dbias.dtype != torch.float32 or dbias.numel() != cols or not dbias.is_contiguous():
        raise ValueError("dbias must be contiguous fp32 [cols]")
    ws = torch.empty(nat.value("eth_bias_gelu_bwd_workspace", rows, cols), dtype=torch.float32, device=x.device)
    nat.call("eth_bias_gelu_bwd_dbias", nat.ptr(dy), nat.ptr(x), nat.ptr(bias), nat.ptr(dx), nat.ptr(dbias),
             nat.ptr(ws), rows, cols, 1 if accumulate else 0, code, nat.stream_ptr(x.device))
    return dx


def bias_dropout_add_fwd(x, bias, residual, p=0.0, seed=0):
    code = _check_half(x, bias, residual)
    rows, cols = _rows_cols(x)
    if residual.shape != x.shape or not residual.is_contiguous() or bias.numel() != cols:
        raise ValueError("shape mismatch")
    out = torch.empty_like(x)
    nat.call("eth_bias_dropout_add_fwd", nat.ptr(x), nat.ptr(bias), nat.ptr(residual), nat.ptr(out), rows, cols,
             float(p), int(seed) & (2**64 - 1), code, nat.stream_ptr(x.device))
    return out


def bias_dropout_add_layer_norm_fwd(x, bias, residual, gamma, beta, p=0.0, seed=0, eps=1e-5):
    """(h, y, mean, rstd): h = bias_dropout_add_fwd(x, bias, residual, p,
    seed) and (y, mean, rstd) = layer_norm_fwd(h, gamma, beta, eps), bit for
    bit, from one kernel that does not read h back."""
    code = _check_half(x, bias, residual, gamma, beta)
    rows, cols = _rows_cols(x)
    if residual.shape != x.shape or not residual.is_contiguous() or bias.numel() != cols:
        raise ValueError("shape mismatch")
    if gamma.numel() != cols or beta.numel() != cols:
        raise ValueError("gamma/beta must match the normalized size")
    h = torch.empty_like(x)
    y = torch.empty_like(x)
    mean = torch.empty(rows, dtype=torch.float32, device=x.device)
    rstd = torch.empty(rows, dtype=torch.float32, device=x.device)
    nat.call("eth_bda_ln_fwd", nat.ptr(x), nat.ptr(bias), nat.ptr(residual), nat.ptr(h), nat.ptr(gamma),
             nat.ptr(beta), nat.ptr(y), nat.ptr(mean), nat.ptr(rstd), rows, cols, float(p),
             int(seed) & (2**64 - 1), float(eps), code, nat.stream_ptr(x.device))
    return h, y, mean, rstd


def dropout_bwd(dy, p, seed):
    code = _check_half(dy)
    rows, cols = _rows_cols(dy)
    dx = torch.empty_like(dy)
    nat.call("eth_dropout_bwd", nat.ptr(dy), nat.ptr(dx), rows, cols, float(p), int(seed) & (2**64 - 1), code,
             nat.stream_ptr(dy.device))
    return dx


def col_sum(x, out, accumulate):
    """out[c] (+)= sum over rows of x[..., c] (fp32 out)."""
    code = _check_half(x)
    rows, cols = _rows_cols(x)
    if out.dtype != torch.float32 or out.numel() != cols or not out.is_contiguous():
        raise ValueError("out must be contiguous fp32 [cols]")
    ws = torch.empty(nat.value("eth_col_sum_workspace", rows, cols), dtype=torch.float32, device=x.device)
    nat.call("eth_col_sum", nat.ptr(x), cols, rows, cols, nat.ptr(out), nat.ptr(ws), 1 if accumulate else 0, code,
             nat.stream_ptr(x.device))
    return out


# ---------------------------------------------------------------- attention --
def _sbhd_strides(t):
    """(seq, batch, head) strides of a [s, b, np, hn] view with hn contiguous."""
    if t.dim() != 4 or t.stride(3) != 1:
        raise ValueError("attention operands must be [s, b, np, hn] views with hn contiguous")
    return (t.stride(0), t.stride(1), t.stride(2))


def _attn_desc(q, dtype_code):
    s, b, n, d = q.shape
    desc = nat.AttnDesc()
    desc.batch, desc.heads, desc.seq, desc.head_dim, desc.dtype = b, n, s, d, dtype_code
    return desc


def attention_fwd(q, k, v, out=None):
    """Causal attention on [s, b, np, hn] views (any seq/batch/head strides).
    Returns (out [s, b, np, hn] view of a contiguous [s, b, np*hn], lse)."""
    code = _check_half(q, k, v)
    if not (q.shape == k.shape == v.shape):
        raise ValueError("q, k, v shapes differ")
    s, b, n, d = q.shape
    if d % 8 or not 8 <= d <= 128 or s < 1:
        raise ValueError(f"attention needs head_dim a multiple of 8 in [8, 128] and seq >= 1 (got {d}, {s})")
    if out is None:
        out = torch.empty(s, b, n * d, dtype=q.dtype, device=q.device)
    o4 = out.view(s, b, n, d)
    lse = torch.empty(b * n, s, dtype=torch.float32, device=q.device)
    desc = _attn_desc(q, code)
    desc.q_strides[:] = _sbhd_strides(q)
    desc.k_strides[:] = _sbhd_strides(k)
    desc.v_strides[:] = _sbhd_strides(v)
    desc.o_strides[:] = _sbhd_strides(o4)
    flops = 2.0 * b * n * s * s * d  # QK^T and PV over the causal half
    _observe("attn_fwd", "begin", flops)
    nat.call("eth_attn_fwd", ctypes.byref(desc), nat.ptr(q), nat.ptr(k), nat.ptr(v), nat.ptr(o4), nat.ptr(lse),
             nat.stream_ptr(q.device))
    _observe("attn_fwd", "end", flops)
    return out, lse


def attention_bwd(q, k, v, out, dout, lse, dq, dk, dv):
    """Gradients of causal attention into dq/dk/dv ([s, b, np, hn] views, e.g.
    of one [s, b, np, 3*hn] buffer).  out/dout are [s, b, np*hn]."""
    code = _check_half(q, k, v, out, dout, dq, dk, dv)
    s, b, n, d = q.shape
    o4 = out.view(s, b, n, d)
    do4 = dout.reshape(s, b, n, d) if dout.is_contiguous() else None
    if do4 is None:
        raise ValueError("dout must be contiguous [s, b, np*hn]")
    if lse.shape != (b * n, s):
        raise ValueError("lse shape mismatch")
    delta = torch.empty(b * n, s, dtype=torch.float32, device=q.device)
    desc = _attn_desc(q, code)
    for name, t in (("q", q), ("k", k), ("v", v), ("o", o4), ("do", do4), ("dq", dq), ("dk", dk), ("dv", dv)):
        if t.shape != q.shape:
            raise ValueError(f"{name} shape mismatch")
        getattr(desc, f"{name}_strides")[:] = _sbhd_strides(t)
    flops = 2.5 * 2.0 * b * n * s * s * d  # dS = dP, dQ, dK, dV: 2.5x the forward's products
    _observe("attn_bwd", "begin", flops)
    nat.call("eth_attn_bwd", ctypes.byref(desc), nat.ptr(q), nat.ptr(k), nat.ptr(v), nat.ptr(o4), nat.ptr(do4),
             nat.ptr(lse), nat.ptr(delta), nat.ptr(dq), nat.ptr(dk), nat.ptr(dv), nat.stream_ptr(q.device))
    _observe("attn_bwd", "end", flops)


def _launch(index, name, *args):
    """nat.call(name, *args, the current stream) on device `index`, whichever
    the current one is."""
    if index == torch._C._cuda_getDevice():
        nat.call(name, *args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            nat.call(name, *args, torch._C._cuda_getCurrentRawStream(index))


def _check_device(index, *ts):
    for t in ts:
        if t.get_device() != index:
            raise ValueError(f"tensors on cuda:{index} and {t.device}: one GPU is needed (no CPU fallback)")


def _thd_strides(name, t, written=False):
    """(row, head) strides of a [rows, heads, hn] view with hn contiguous."""
    rows, heads, hn = t.shape
    sr, sh, sd = t.stride()
    if hn > 1 and sd != 1:
        raise ValueError(f"{name} must be a [rows, heads, hn] view with hn contiguous")
    # (the stride of a dimension of size 1 means nothing and may be anything)
    sr, sh = sr if rows > 1 else heads * hn, sh if heads > 1 else hn
    if sr % 8 or sh % 8:
        raise ValueError(f"{name}: rows must be 16-byte aligned")
    if written and not (sh >= hn and sr >= (heads - 1) * sh + hn or sr >= hn and sh >= (rows - 1) * sr + hn):
        raise ValueError(f"{name}: rows that are written may not overlap")
    return sr, sh


def _packed_desc(packed, scale, q, k, v, *grads):
    """(descriptor, its reference, workspace bytes) of a packed attention call,
    built and checked once for these types, shapes and strides and kept with
    the plan (the addresses are the call's; the entry checks their alignment)."""
    scale = None if scale is None else float(scale)
    key = (scale, *[x for t in (q, k, v, *grads) for x in (t.shape, t.stride(), t.dtype)])
    got = packed.descriptors.get(key)
    if got is not None:
        return got
    code = _HALF_CODES.get(q.dtype)
    if code is None or any(t.dtype != q.dtype for t in (k, v, *grads)):
        raise ValueError(f"packed attention needs bf16 or fp16 tensors of one type, got "
                         f"{', '.join(str(t.dtype) for t in (q, k, v, *grads))}")
    if q.dim() != 3 or k.dim() != 3 or v.shape != k.shape:
        raise ValueError("packed attention needs q [rows, heads, hn] and k, v [rows, kv_heads, hn]")
    rows, n, d = q.shape
    m = k.shape[1]
    if k.shape[0] != rows or k.shape[2] != d or rows != packed.total:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and {packed.total} packed rows do not match")
    if d % 8 or not 8 <= d <= 128:
        raise ValueError(f"packed attention needs head_dim a multiple of 8 in [8, 128] (got {d})")
    if m < 1 or n < 1 or n % m:
        raise ValueError(f"{n} query heads cannot share {m} key and value heads")
    c = d**-0.5 if scale is None else scale
    if not 2.0**-100 <= c <= 2.0**100:
        raise ValueError(f"scale must be positive and finite (got {scale})")
    desc = nat.PackedAttnDesc()
    desc.rows, desc.heads, desc.kv_heads, desc.head_dim, desc.dtype, desc.scale = rows, n, m, d, code, c
    (desc.q_tiles, desc.n_q_tiles, desc.k_tiles, desc.n_k_tiles, desc.q_split[:], desc.k_split[:]) = packed.plan(
        n, m, d)
    for name, t in (("q", q), ("k", k), ("v", v)):
        getattr(desc, f"{name}_strides")[:] = _thd_strides(name, t)
    desc.o_strides[:] = desc.do_strides[:] = (n * d, d)  # (contiguous [rows, n*hn])
    for name, t, like in zip(("dq", "dk", "dv"), grads, (q, k, v)):
        if t.shape != like.shape:
            raise ValueError(f"{name} shape mismatch")
        getattr(desc, f"{name}_strides")[:] = _thd_strides(name, t, written=True)
    ref = ctypes.byref(desc)
    size = 0
    if desc.q_split[0] or grads and desc.k_split[0]:
        size = nat.value("eth_packed_attn_workspace", ref, 1 if grads else 0)
    got = packed.descriptors[key] = desc, ref, size
    return got


def _packed_flops(packed, n, d):
    return 2.0 * n * d * sum(x * (x + 1) for x in packed.lengths)  # QK^T and PV over the causal half


def _packed_launch(name, kind, work, q, packed, *args):
    packed.in_use()
    if _observer is None:
        return _launch(packed.device.index, name, *args)
    flops = work * _packed_flops(packed, q.shape[1], q.shape[2])
    _observe(kind, "begin", flops)
    _launch(packed.device.index, name, *args)
    _observe(kind, "end", flops)


def packed_attention_fwd(q, k, v, packed, scale=None, out=None):
    """Causal attention over `packed` (PackedSequences) of q [rows, n, hn] and
    k, v [rows, m, hn] views with any row and head strides; query head h reads
    key/value head h // (n // m).  Returns (out [rows, n*hn], lse [n, rows],
    log2 domain); rows of no sequence get zeros (lse -inf).  A given `out` shares
    no memory with q, k and v."""
    _check_device(packed.device.index, q, k, v)
    _, ref, size = _packed_desc(packed, scale, q, k, v)
    rows, n, d = q.shape
    if out is None:
        out = torch.empty(rows, n * d, dtype=q.dtype, device=q.device)
    elif out.shape != (rows, n * d) or out.dtype != q.dtype or out.device != q.device or not out.is_contiguous():
        raise ValueError("out must be a contiguous [rows, n*hn] tensor like q")
    lse = torch.empty(n, rows, dtype=torch.float32, device=q.device)
    ws = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None
    _packed_launch("eth_packed_attn_fwd", "attn_fwd", 1.0, q, packed, ref, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                   out.data_ptr(), lse.data_ptr(), nat.ptr(ws))
    return out, lse


def packed_attention_bwd(q, k, v, out, dout, lse, packed, dq, dk, dv, scale=None):
    """Gradients of packed_attention_fwd into dq [rows, n, hn] and dk, dv
    [rows, m, hn] views; out / dout are contiguous [rows, n*hn].  dk and dv are
    summed over the query heads that share them, in a fixed order; rows of no
    sequence get zeros.  dq, dk and dv share no memory with each other or with the
    other operands."""
    _check_device(packed.device.index, q, k, v, out, dout, lse, dq, dk, dv)
    desc = _packed_desc(packed, scale, q, k, v, dq, dk, dv)
    rows, n, d = q.shape
    for name, t in (("out", out), ("dout", dout)):
        if t.shape != (rows, n * d) or t.dtype != q.dtype or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous [rows, n*hn] like q")
    if lse.shape != (n, rows) or lse.dtype != torch.float32 or not lse.is_contiguous():
        raise ValueError("lse must be the forward's fp32 [n, rows]")
    _packed_bwd(desc, q, k, v, out, dout, lse, packed, dq, dk, dv)


def _packed_bwd(desc, q, k, v, out, dout, lse, packed, dq, dk, dv):
    _, ref, size = desc
    delta = torch.empty(lse.shape, dtype=torch.float32, device=q.device)
    ws = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None
    _packed_launch("eth_packed_attn_bwd", "attn_bwd", 2.5, q, packed, ref, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                   out.data_ptr(), dout.data_ptr(), lse.data_ptr(), delta.data_ptr(), dq.data_ptr(), dk.data_ptr(),
                   dv.data_ptr(), nat.ptr(ws))


def _packed_attention_grads(q, k, v, out, dout, lse, packed, scale=None):
    """(dq, dk, dv) of packed_attention_bwd in new tensors, for the very q, k,
    v, out, lse and scale of a packed_attention_fwd call, which are not checked
    again but for where and how they lie now (hooks on saved tensors may have
    moved them); dout is like out."""
    _check_device(packed.device.index, q, k, v, out, lse)
    if out.dtype != q.dtype or lse.dtype != torch.float32 or not out.is_contiguous() or not lse.is_contiguous():
        raise ValueError("saved tensors came back in another type or layout")
    key = "grads", scale, q.shape, q.stride(), k.shape, k.stride(), v.stride(), q.dtype, k.dtype, v.dtype
    desc = packed.descriptors.get(key)
    dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    dk = torch.empty(k.shape, dtype=q.dtype, device=q.device)
    dv = torch.empty(k.shape, dtype=q.dtype, device=q.device)
    if desc is None:
        desc = packed.descriptors[key] = _packed_desc(packed, scale, q, k, v, dq, dk, dv)
    if dout.shape != out.shape or dout.dtype != out.dtype or dout.get_device() != out.get_device():
        raise ValueError("dout must be like out")
    dout = dout.contiguous()
    if dout.data_ptr() % 16:  # (a part of what autograd cut up: its rows start where the part does)
        dout = dout.clone()
    _packed_bwd(desc, q, k, v, out, dout, lse, packed, dq, dk, dv)
    return dq, dk, dv


# --------------------------------------------------------------- vocabulary --
def _check_ids(t, shape=None):
    if t.dtype != torch.int64 or not t.is_contiguous() or not t.is_cuda:
        raise ValueError("token / position ids must be contiguous int64 GPU tensors")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"ids shape {tuple(t.shape)} != {tuple(shape)}")


def embedding_fwd(tokens, positions, word, pos, bad_flag):
    """[b, s] ids -> [s, b, h] = word[tokens] + pos[positions] (16-bit)."""
    code = _check_half(word, pos)
    b, s = tokens.shape
    _check_ids(tokens)
    _check_ids(positions, (b, s))
    V, h = word.shape
    P, h2 = pos.shape
    if h != h2 or not word.is_contiguous() or not pos.is_contiguous():
        raise ValueError("embedding tables must be contiguous [rows, hidden] with equal hidden")
    out = torch.empty(s, b, h, dtype=word.dtype, device=word.device)
    nat.call("eth_embedding_fwd", nat.ptr(tokens), nat.ptr(positions), nat.ptr(word), nat.ptr(pos), nat.ptr(out),
             b, s, h, V, P, nat.ptr(bad_flag), code, nat.stream_ptr(word.device))
    return out


def embedding_bwd(tokens, positions, dout, dword, dpos):
    """fp32 dword[tokens] += dout and dpos[positions] += dout (dout [s, b, h]),
    bitwise deterministic (sorted ids, one owner per table row)."""
    code = _check_half(dout)
    b, s = tokens.shape
    _check_ids(tokens)
    _check_ids(positions, (b, s))
    if dout.shape[:2] != (s, b) or not dout.is_contiguous():
        raise ValueError("dout must be contiguous [s, b, h]")
    h = dout.shape[2]
    for t in (dword, dpos):
        if t is not None and (t.dtype != torch.float32 or t.shape[1] != h or not t.is_contiguous()):
            raise ValueError("embedding gradients must be contiguous fp32 [rows, hidden]")
    V = dword.shape[0] if dword is not None else 1
    P = dpos.shape[0] if dpos is not None else 1
    # (the call's own: its two launches may have another thread's between them)
    ws = torch.empty(nat.value("eth_embedding_bwd_workspace", b, s), dtype=torch.uint8, device=dout.device)
    nat.call("eth_embedding_bwd", nat.ptr(tokens), nat.ptr(positions), nat.ptr(dout), nat.ptr(dword), nat.ptr(dpos),
             nat.ptr(ws), b, s, h, V, P, code, nat.stream_ptr(dout.device))


def xent_fwd(logits2d, labels, bad_flag):
    """Per-row loss and lse (fp32) of 16-bit logits [rows, V]."""
    code = _check_half(logits2d)
    rows, V = logits2d.shape
    if logits2d.stride(1) != 1:
        raise ValueError("logits rows must be contiguous")
    _check_ids(labels, (rows,))
    loss = torch.empty(rows, dtype=torch.float32, device=logits2d.device)
    lse = torch.empty(rows, dtype=torch.float32, device=logits2d.device)
    nat.call("eth_xent_fwd", nat.ptr(logits2d), logits2d.stride(0), nat.ptr(labels), nat.ptr(loss), nat.ptr(lse),
             rows, V, nat.ptr(bad_flag), code, nat.stream_ptr(logits2d.device))
    return loss, lse


def xent_bwd(logits2d, labels, lse, dloss):
    code = _check_half(logits2d)
    rows, V = logits2d.shape
    if dloss.dtype != torch.float32 or dloss.numel() != rows or not dloss.is_contiguous():
        raise ValueError("dloss must be contiguous fp32 [rows]")
    dz = torch.empty(rows, V, dtype=logits2d.dtype, device=logits2d.device)
    nat.call("eth_xent_bwd", nat.ptr(logits2d), logits2d.stride(0), nat.ptr(labels), nat.ptr(lse), nat.ptr(dloss),
             nat.ptr(dz), V, rows, V, code, nat.stream_ptr(logits2d.device))
    return dz


def _check_logits(logits2d, bad_flag, *ts):
    """(device index, dtype code, rows, V, row stride) of [rows, V] logits in
    any of the three types."""
    if logits2d.dim() != 2 or logits2d.shape[1] < 1:
        raise ValueError("logits must be [rows, V]")
    index = logits2d.get_device()
    if index < 0:
        raise ValueError("eth_amd kernels run on the GPU only (no CPU fallback)")
    code = nat.dtype_code(logits2d.dtype)
    rows, V = logits2d.shape
    ld, s1 = logits2d.stride()
    if V > 1 and s1 != 1:
        raise ValueError("logits rows must be contiguous")
    if rows <= 1:
        ld = V
    if ld < V:
        raise ValueError("logits rows may not overlap")
    if bad_flag.dtype != torch.int32 or bad_flag.numel() < 1:
        raise ValueError("bad_flag must be an int32 tensor")
    _check_device(index, bad_flag, *ts)
    return index, code, rows, V, ld


def _saved_layout(layout, logits2d, *ts):
    """The layout of logits that a forward checked (`layout`: _check_logits'
    result), as autograd gives them back to its backward: hooks on saved tensors
    may have moved them, and rows that were apart then lie side by side.  `ts`:
    (tensor, type) of what was contiguous beside them."""
    index, code, rows, V, _ = layout
    ld, s1 = logits2d.stride()
    if rows <= 1:
        ld = V
    if (logits2d.shape != (rows, V) or nat.dtype_code(logits2d.dtype) != code or V > 1 and s1 != 1 or ld < V
            or logits2d.get_device() != index):
        raise ValueError("saved logits came back in another shape, type or layout, or elsewhere")
    for t, dtype in ts:
        if t.dtype != dtype or not t.is_contiguous() or t.get_device() != index:
            raise ValueError("saved tensors came back in another type or layout, or elsewhere")
    return index, code, rows, V, ld


def _check_row_values(name, t, rows):
    if t.dtype != torch.float32 or t.shape != (rows,) or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous fp32 [rows]")


def _check_stats(stats, rows, n):
    if stats.dtype != torch.float32 or stats.shape != (rows, n) or not stats.is_contiguous():
        raise ValueError(f"stats must be the forward's fp32 [rows, {n}]")


def token_logprobs_fwd(logits2d, tokens, top_k, bad_flag, ignore_index=-100):
    """(logprob [rows], entropy [rows], stats [rows, 2], top_logprobs [rows,
    top_k] fp32, top_ids [rows, top_k] int64) of logits [rows, V] in bf16, fp16
    or fp32: the log probability of each row's token, the row's entropy and its
    top_k largest log probabilities, equal ones by the lowest id.  Rows with
    token `ignore_index` give 0, 0, -inf and -1; other ids outside the
    vocabulary are clamped and flagged in `bad_flag`."""
    return _token_logprobs_fwd(logits2d, tokens, top_k, bad_flag, ignore_index, (logits2d.shape[0],))[:5]


def _token_logprobs_fwd(logits2d, tokens, top_k, bad_flag, ignore_index, shape):
    """token_logprobs_fwd with the rows in `shape` in its results, and behind
    them the operands' layout for the backward."""
    layout = index, code, rows, V, ld = _check_logits(logits2d, bad_flag, tokens)
    top_k, ignore_index = operator.index(top_k), operator.index(ignore_index)
    _check_ids(tokens, (rows,))
    if not 0 <= top_k <= min(128, V):
        raise ValueError(f"top_k must be in [0, 128] and within the vocabulary (got {top_k})")
    new = functools.partial(torch.empty, dtype=torch.float32, device=logits2d.device)
    logprob, entropy, stats, top = new(shape), new(shape), new(rows, 2), new(*shape, top_k)
    ids = torch.empty(*shape, top_k, dtype=torch.int64, device=logits2d.device)
    if rows:
        # (the call's own: its two launches may have another thread's between them)
        ws = nat.value("eth_token_logprobs_workspace", rows, V, top_k, code)
        ws = torch.empty(ws, dtype=torch.uint8, device=logits2d.device) if ws else None
        _launch(index, "eth_token_logprobs_fwd", logits2d.data_ptr(), ld, tokens.data_ptr(), ignore_index,
                logprob.data_ptr(), entropy.data_ptr(), stats.data_ptr(), top.data_ptr(), ids.data_ptr(), top_k,
                nat.ptr(ws), rows, V, bad_flag.data_ptr(), code)
    return logprob, entropy, stats, top, ids, layout


def token_logprobs_bwd(logits2d, tokens, stats, entropy, dlogprob, dentropy, bad_flag, ignore_index=-100):
    """dlogits [rows, V] for upstream gradients of logprob and entropy (fp32
    [rows]; one of them may be None)."""
    given = [t for t in (dlogprob, dentropy) if t is not None]
    index, code, rows, V, ld = _check_logits(logits2d, bad_flag, tokens, stats, entropy, *given)
    _check_ids(tokens, (rows,))
    _check_stats(stats, rows, 2)
    for name, t in (("entropy", entropy), ("dlogprob", dlogprob), ("dentropy", dentropy)):
        if t is not None:
            _check_row_values(name, t, rows)
    if not given:
        raise ValueError("token_logprobs_bwd needs dlogprob or dentropy")
    return _token_logprobs_bwd((index, code, rows, V, ld), logits2d, tokens, stats, entropy, dlogprob, dentropy,
                               ignore_index, logits2d.shape)


def _token_logprobs_bwd(layout, logits2d, tokens, stats, entropy, dlogprob, dentropy, ignore_index, shape):
    """token_logprobs_bwd of operands that a forward checked (`layout`: their
    layout now; upstream gradients as contiguous fp32 [rows])."""
    index, code, rows, V, ld = layout
    dz = torch.empty(shape, dtype=logits2d.dtype, device=logits2d.device)
    if rows:
        _launch(index, "eth_token_logprobs_bwd", logits2d.data_ptr(), ld, tokens.data_ptr(), operator.index(ignore_index),
                stats.data_ptr(), entropy.data_ptr(), nat.ptr(dlogprob), nat.ptr(dentropy), dz.data_ptr(), V, rows, V,
                code)
    return dz


def _check_teacher(teacher_ids, teacher_logits, rows, temperature):
    if teacher_ids.dim() != 2 or teacher_logits.shape != teacher_ids.shape:
        raise ValueError("teacher ids and logits must both be [rows, k]")
    k = teacher_ids.shape[1]
    if not 1 <= k <= 256:
        raise ValueError(f"1 to 256 teacher entries a row are needed (got {k})")
    _check_ids(teacher_ids, (rows, k))
    if not teacher_logits.is_contiguous():
        raise ValueError("teacher logits must be contiguous")
    if not 2.0**-20 <= temperature <= 2.0**20:
        raise ValueError(f"temperature must be positive and finite (got {temperature})")
    return k, nat.dtype_code(teacher_logits.dtype)


def topk_distill_fwd(logits2d, teacher_ids, teacher_logits, temperature, bad_flag):
    """(loss [rows], stats [rows, 4]): temperature^2 * sum q (log q - log p[id])
    with q the softmax of a row's k teacher logits (any of the three types) and
    p that of its V logits, both at the temperature.  Negative ids and teacher
    logits of -inf are no entries; ids past the vocabulary are none either and
    are flagged in `bad_flag`."""
    return _topk_distill_fwd(logits2d, teacher_ids, teacher_logits, temperature, bad_flag, (logits2d.shape[0],))[:2]


def _topk_distill_fwd(logits2d, teacher_ids, teacher_logits, temperature, bad_flag, shape):
    """topk_distill_fwd with the rows in `shape` in its loss, and behind its
    results the operands' layout for the backward."""
    layout = index, code, rows, V, ld = _check_logits(logits2d, bad_flag, teacher_ids, teacher_logits)
    k, teacher_code = _check_teacher(teacher_ids, teacher_logits, rows, temperature)
    loss = torch.empty(shape, dtype=torch.float32, device=logits2d.device)
    stats = torch.empty(rows, 4, dtype=torch.float32, device=logits2d.device)
    if rows:
        ws = nat.value("eth_topk_distill_workspace", rows, V, code)
        ws = torch.empty(ws, dtype=torch.uint8, device=logits2d.device) if ws else None
        _launch(index, "eth_topk_distill_fwd", logits2d.data_ptr(), ld, teacher_ids.data_ptr(),
                teacher_logits.data_ptr(), teacher_code, k, float(temperature), loss.data_ptr(), stats.data_ptr(),
                nat.ptr(ws), rows, V, bad_flag.data_ptr(), code)
    return loss, stats, layout


def topk_distill_bwd(logits2d, teacher_ids, teacher_logits, temperature, stats, dloss, bad_flag):
    """dlogits [rows, V] of topk_distill_fwd's loss (dloss fp32 [rows])."""
    index, code, rows, V, ld = _check_logits(logits2d, bad_flag, teacher_ids, teacher_logits, stats, dloss)
    _check_teacher(teacher_ids, teacher_logits, rows, temperature)
    _check_stats(stats, rows, 4)
    _check_row_values("dloss", dloss, rows)
    return _topk_distill_bwd((index, code, rows, V, ld), logits2d, teacher_ids, teacher_logits, temperature, stats,
                             dloss, bad_flag, logits2d.shape)


def _topk_distill_bwd(layout, logits2d, teacher_ids, teacher_logits, temperature, stats, dloss, bad_flag, shape):
    """topk_distill_bwd of operands that a forward checked (`layout`: their
    layout now; dloss as contiguous fp32 [rows])."""
    index, code, rows, V, ld = layout
    k, teacher_code = teacher_ids.shape[1], nat.dtype_code(teacher_logits.dtype)
    dz = torch.empty(shape, dtype=logits2d.dtype, device=logits2d.device)
    if rows:
        _launch(index, "eth_topk_distill_bwd", logits2d.data_ptr(), ld, teacher_ids.data_ptr(),
                teacher_logits.data_ptr(), teacher_code, k, float(temperature), stats.data_ptr(), dloss.data_ptr(),
                dz.data_ptr(), V, rows, V, bad_flag.data_ptr(), code)
    return dz


def _check_head(hidden2d, weight, labels, *ts):
    """(device index, dtype code, rows, H, V, row strides) of a linear head's
    operands: hidden [rows, H], weight [V, H], labels [rows]."""
    if hidden2d.dim() != 2 or weight.dim() != 2 or hidden2d.shape[1] != weight.shape[1] or weight.shape[0] < 1:
        raise ValueError(f"hidden {tuple(hidden2d.shape)} and weight {tuple(weight.shape)} must be [rows, H] and [V, H]")
    code = _HALF_CODES.get(hidden2d.dtype)
    if code is None or weight.dtype != hidden2d.dtype:
        raise ValueError(f"hidden and weight must be bf16 or fp16 and of one type, got {hidden2d.dtype}, {weight.dtype}")
    index = hidden2d.get_device()
    if index < 0:
        raise ValueError("eth_amd kernels run on the GPU only (no CPU fallback)")
    _check_device(index, weight, labels, *ts)
    rows, H = hidden2d.shape
    V = weight.shape[0]
    if H < 1 or H % 8:
        raise ValueError(f"the hidden size must be a multiple of 8 (got {H})")
    _check_ids(labels, (rows,))
    strides = []
    for name, t in (("hidden", hidden2d), ("weight", weight)):
        ld, s1 = t.stride()
        if s1 != 1:
            raise ValueError(f"{name} rows must be contiguous")
        ld = H if t.shape[0] <= 1 else ld
        if ld < H or ld % 8 or t.data_ptr() % 16:
            raise ValueError(f"{name}: rows must be 16-byte aligned and may not overlap")
        strides.append(ld)
    return index, code, rows, H, V, *strides


def linear_xent_fwd(hidden2d, weight, labels, bad_flag, ignore_index=-100):
    """(loss [rows], lse [2, rows]) in fp32 of the cross entropy of logits hidden2d
    [rows, H] @ weight[V, H]^T, which are not kept, against int64 labels [rows]; lse,
    for the backward, is the logits' logsumexp (log2 domain) and the loss again.
    Rows with label `ignore_index` have loss 0 and are not read; other labels
    outside the vocabulary are clamped and flagged in `bad_flag`."""
    index, code, rows, H, V, ldh, ldw = _check_head(hidden2d, weight, labels, bad_flag)
    if bad_flag.dtype != torch.int32 or bad_flag.numel() < 1:
        raise ValueError("bad_flag must be an int32 tensor")
    loss = torch.empty(rows, dtype=torch.float32, device=hidden2d.device)
    lse = torch.empty(2, rows, dtype=torch.float32, device=hidden2d.device)
    if rows:
        ws = nat.value("eth_linear_xent_workspace", rows, H, V, ldw, 0)
        ws = torch.empty(ws, dtype=torch.uint8, device=hidden2d.device)
        _launch(index, "eth_linear_xent_fwd", hidden2d.data_ptr(), ldh, weight.data_ptr(), ldw, labels.data_ptr(),
                operator.index(ignore_index), loss.data_ptr(), lse.data_ptr(), ws.data_ptr(), rows, H, V,
                bad_flag.data_ptr(), code)
    return loss, lse


def linear_xent_bwd(hidden2d, weight, labels, lse, dloss, ignore_index=-100, need_dhidden=True, need_dweight=True,
                    dweight=None, accumulate=False):
    """(dhidden [rows, H], dweight [V, H]) for dloss fp32 [rows], None where not
    needed: in the operands' type, or dweight into a given fp32 tensor, stored or
    added."""
    index, code, rows, H, V, ldh, ldw = _check_head(hidden2d, weight, labels, lse, dloss)
    if lse.dtype != torch.float32 or lse.shape != (2, rows) or not lse.is_contiguous():
        raise ValueError("lse must be the forward's fp32 [2, rows]")
    _check_row_values("dloss", dloss, rows)
    if dweight is not None:
        _check_device(index, dweight)
        if dweight.dtype != torch.float32 or dweight.shape != (V, H) or not dweight.is_contiguous():
            raise ValueError("dweight must be contiguous fp32 [V, H]")
        if dweight.data_ptr() % 16:
            raise ValueError("dweight must be 16-byte aligned")
        need_dweight = True
    elif accumulate:
        raise ValueError("accumulate needs a given dweight")
    elif need_dweight:
        dweight = torch.empty(V, H, dtype=weight.dtype, device=weight.device)
    dhidden = torch.empty(rows, H, dtype=hidden2d.dtype, device=hidden2d.device) if need_dhidden else None
    if not rows:
        if need_dweight and not accumulate:
            dweight.zero_()
    elif need_dhidden or need_dweight:
        ws = nat.value("eth_linear_xent_workspace", rows, H, V, ldw, (1 if need_dhidden else 0) + (2 if need_dweight else 0))
        ws = torch.empty(ws, dtype=torch.uint8, device=hidden2d.device)
        _launch(index, "eth_linear_xent_bwd", hidden2d.data_ptr(), ldh, weight.data_ptr(), ldw, labels.data_ptr(),
                operator.index(ignore_index), lse.data_ptr(), dloss.data_ptr(), nat.ptr(dhidden), nat.ptr(dweight),
                nat.dtype_code(dweight.dtype) if need_dweight else code, 1 if accumulate else 0, ws.data_ptr(), rows, H,
                V, code)
    return dhidden, dweight


def _adapter_desc(x2d, weight, lora_a, lora_b, rows, *ts):
    """(device index, descriptor) of an adapted projection's operands, for the
    rows of `rows` (AdapterRows)."""
    index = rows.device.index
    _check_device(index, x2d, weight, lora_a, lora_b, *ts)
    code = _HALF_CODES.get(x2d.dtype)
    if code is None or any(t.dtype != x2d.dtype for t in (weight, lora_a, lora_b)):
        raise ValueError(f"adapted projections need bf16 or fp16 tensors of one type, got "
                         f"{', '.join(str(t.dtype) for t in (x2d, weight, lora_a, lora_b))}")
    if x2d.dim() != 2 or weight.dim() != 2 or lora_a.dim() != 3 or lora_b.dim() != 3:
        raise ValueError("x [rows, in], weight [out, in], lora_a [adapters, r, in] and lora_b [adapters, out, r] are needed")
    M, K = x2d.shape
    N = weight.shape[0]
    adapters, r, _ = lora_a.shape
    if weight.shape[1] != K or lora_a.shape[2] != K or lora_b.shape != (adapters, N, r) or M != rows.total:
        raise ValueError(f"x {tuple(x2d.shape)}, weight {tuple(weight.shape)}, lora_a {tuple(lora_a.shape)}, lora_b "
                         f"{tuple(lora_b.shape)} and {rows.total} rows do not match")
    if K < 1 or N < 1 or K % 8 or N % 8:
        raise ValueError(f"in and out must be multiples of 8 (got {K}, {N})")
    if not 8 <= r <= 128 or r % 8:
        raise ValueError(f"the rank must be a multiple of 8 up to 128 (got {r})")
    if rows.n_listed > adapters or not 0 < adapters < 65536:
        raise ValueError(f"rows use adapter {rows.n_listed - 1} of {adapters}")
    desc = nat.AdapterDesc()
    strides = []
    for name, t in (("x", x2d), ("weight", weight)):
        ld, s1 = t.stride()
        ld = K if t.shape[0] <= 1 else ld
        if s1 != 1 or ld < K or ld % 8 or t.data_ptr() % 16:
            raise ValueError(f"{name}: rows must be contiguous, 16-byte aligned and apart")
        strides.append(ld)
    for name, t in (("lora_a", lora_a), ("lora_b", lora_b)):
        if not t.is_contiguous() or t.data_ptr() % 16:
            raise ValueError(f"{name} must be contiguous and 16-byte aligned")
    desc.rows, desc.in_, desc.out, desc.ldx, desc.ldw = M, K, N, *strides
    desc.tiles, desc.chunks, desc.first_chunk, desc.used, desc.of_row = rows.addresses
    desc.n_tiles, desc.n_chunks, desc.n_used, desc.n_listed = rows.n_tiles, rows.n_chunks, rows.n_used, rows.n_listed
    desc.adapters, desc.rank, desc.dtype = adapters, r, code
    return index, desc


def _adapter_workspace(desc, backward, device):
    size = nat.value("eth_adapter_linear_workspace", ctypes.byref(desc), backward)
    if size < 0:
        raise ValueError(nat.load().eth_last_error().decode(errors="replace"))
    return torch.empty(size, dtype=torch.uint8, device=device)


def adapter_linear_fwd(x2d, weight, bias, lora_a, lora_b, rows, save=False):
    """(y [rows, out], saved): y = x2d weight^T + bias + scale (x2d A^T) B^T with
    each row's adapter (A [r, in] and B [out, r] of lora_a and lora_b) and scale of
    `rows` (AdapterRows); rows of no adapter without the last term.  saved: what
    dB needs, or None without `save`."""
    index, desc = _adapter_desc(x2d, weight, lora_a, lora_b, rows)
    M, N, rp = desc.rows, desc.out, -(-desc.rank // 32) * 32
    if bias is not None:
        _check_device(index, bias)
        if bias.dtype != x2d.dtype or bias.shape != (N,) or not bias.is_contiguous():
            raise ValueError("bias must be a contiguous [out] tensor of the input type")
    new = functools.partial(torch.empty, device=x2d.device)
    y = new(M, N, dtype=x2d.dtype)
    saved = None
    if save:
        saved = (new(rows.n_tiles, rp, nat.ADAPTER_TILE_ROWS, dtype=x2d.dtype),
                 new(rows.n_tiles, dtype=torch.float32))
    ut, tile_scale = saved or (None, None)
    ws = _adapter_workspace(desc, 0, x2d.device)
    rows.in_use()
    _launch(index, "eth_adapter_linear_fwd", ctypes.byref(desc), x2d.data_ptr(), weight.data_ptr(), nat.ptr(bias),
            lora_a.data_ptr(), lora_b.data_ptr(), y.data_ptr(), nat.ptr(ut), nat.ptr(tile_scale), ws.data_ptr())
    return y, saved


def adapter_linear_bwd(x2d, weight, lora_a, lora_b, dy, rows, saved=None, need_dx=True, da=None, db=None):
    """dx [rows, in] (None without need_dx) of adapter_linear_fwd for contiguous dy
    [rows, out].  da, db: pairs (tensor like lora_a / lora_b, in their type or fp32,
    that the gradient is written to, whether it is added, fp32 alone), or None; db
    needs the forward's `saved`.  Adapters without rows get zeros."""
    index, desc = _adapter_desc(x2d, weight, lora_a, lora_b, rows, dy)
    if dy.shape != (desc.rows, desc.out) or dy.dtype != x2d.dtype or not dy.is_contiguous() or dy.data_ptr() % 16:
        raise ValueError("dy must be a contiguous, 16-byte aligned [rows, out] tensor of the input type")
    grads = []
    for name, pair, like in (("da", da, lora_a), ("db", db, lora_b)):
        entry = nat.AdapterGrad()
        if pair is not None:
            t, accumulate = pair
            _check_device(index, t)
            if t.shape != like.shape or t.dtype not in (like.dtype, torch.float32) or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous tensor like its adapters, or fp32")
            if t.data_ptr() % 16 or accumulate and t.dtype != torch.float32:
                raise ValueError(f"{name} must be 16-byte aligned, and fp32 where it is added to")
            entry.grad, entry.fp32, entry.accumulate = t.data_ptr(), t.dtype == torch.float32, bool(accumulate)
        grads.append(entry)
    ut, tile_scale = saved or (None, None)
    if db is not None:
        rp = -(-desc.rank // 32) * 32
        if (saved is None or ut.shape != (rows.n_tiles, rp, nat.ADAPTER_TILE_ROWS) or ut.dtype != x2d.dtype
                or not ut.is_contiguous() or tile_scale.shape != (rows.n_tiles,) or tile_scale.dtype != torch.float32
                or not tile_scale.is_contiguous()):
            raise ValueError("db needs what the forward saved")
        _check_device(index, ut, tile_scale)
    dx = torch.empty(desc.rows, desc.in_, dtype=x2d.dtype, device=x2d.device) if need_dx else None
    if not need_dx and da is None and db is None:
        return None
    ws = _adapter_workspace(desc, 1, x2d.device)
    rows.in_use()
    _launch(index, "eth_adapter_linear_bwd", ctypes.byref(desc), x2d.data_ptr(), weight.data_ptr(), lora_a.data_ptr(),
            lora_b.data_ptr(), dy.data_ptr(), nat.ptr(ut), nat.ptr(tile_scale), nat.ptr(dx), ctypes.byref(grads[0]),
            ctypes.byref(grads[1]), ws.data_ptr())
    return dx


def synthetic_batch(sample_ids, seq, vocab, device):
    """tokens [b, s] int64, loss_mask [b, s] fp32, position_ids [b, s] int64
    of the deterministic synthetic batch, computed on the device in one
    launch per 64 samples (the ids cross as a host array)."""
    if isinstance(sample_ids, torch.Tensor):
        sample_ids = sample_ids.detach().cpu()  # the ids travel to the kernel by value
    ids = np.ascontiguousarray(np.asarray(sample_ids, dtype=np.int64).reshape(-1))
    b = ids.size
    if seq <= 0 or vocab <= 0:
        raise ValueError("sequence length and vocabulary size must be positive")
    tokens = torch.empty(b, seq, dtype=torch.int64, device=device)
    mask = torch.empty(b, seq, dtype=torch.float32, device=device)
    positions = torch.empty(b, seq, dtype=torch.int64, device=device)
    nat.require_cuda(tokens)
    nat.call("eth_synthetic_batch", ids.ctypes.data_as(ctypes.c_void_p), b, seq, vocab, nat.ptr(tokens),
             nat.ptr(mask), nat.ptr(positions), nat.stream_ptr(tokens.device))
    return tokens, mask, positions


def tied_grad_sum(root, copy):
    """root = copy = root + copy (main grads of a tied weight: fp32, or 16-bit
    with the sum rounded once to their dtype)."""
    if root.dtype != copy.dtype or root.shape != copy.shape:
        raise ValueError("tied gradients must be tensors of one dtype and shape")
    if not (root.is_contiguous() and copy.is_contiguous()):
        raise ValueError("tied gradients must be contiguous")
    if root.dtype == torch.float32:
        nat.call("eth_tied_grad_sum", nat.ptr(root), nat.ptr(copy), root.numel(), nat.stream_ptr(root.device))
    else:
        code = _check_half(root, copy)
        nat.call("eth_tied_grad_sum_half", nat.ptr(root), nat.ptr(copy), root.numel(), code,
                 nat.stream_ptr(root.device))
