"""autograd Functions over the HIP kernels.

Weight and bias gradients follow the Megatron local-DDP contract
(eth/runtime/megatron/model/distributed.py:116-123): when a parameter has an
fp32 `main_grad` buffer, its gradient is accumulated straight into it by
the kernel (the wgrad GEMM adds into main_grad; bias / LayerNorm gradients
are reduced in fp32 and added), and the autograd gradient returned for the
parameter is None, so `param.grad` stays None.  Without `main_grad`, or with
a 16-bit one (fp16 training without fp32 accumulation, the reference's
default), the gradient is returned in the parameter's dtype -- rounded once
from its fp32 reduction -- and the DDP hook adds it into main_grad, a second
rounding, as the reference's `main_grad.add_(param.grad)` does.
"""

import threading

import torch

from .. import kernels as K
from .distributed import grad_written, main_grad_target, materialize_main_grad


# open overlapped_wgrad contexts (of every thread) and the stream that the
# first of them was entered on, as (device index, handle)
_overlap = {"wgrad": 0, "home": None}
_overlap_lock = threading.Lock()


def _here(index):
    return index, torch._C._cuda_getCurrentRawStream(index)


def _stream(here):
    index, handle = here
    return torch.cuda.ExternalStream(handle, device=index) if handle else torch.cuda.default_stream(index)


class overlapped_wgrad:
    """Within this context, LinearFn's large weight-gradient GEMMs into
    main_grad run on a side stream, overlapped with the data-gradient chain.
    Small ones (_SIDE_MIN_FLOPS) stay in line where their node runs on the
    stream the context was entered on.  Contributions to one weight are
    ordered whatever streams their nodes run on, and on exit the current
    stream waits for all of them, so the weights' main grads are complete for
    whatever runs next on it.  Contexts entered on different streams without
    a wait between them are the caller's to order."""

    def __enter__(self):
        self._mark = K.side_mark()
        with _overlap_lock:
            if _overlap["wgrad"] == 0 and torch.cuda.is_initialized():
                _overlap["home"] = _here(torch._C._cuda_getDevice())
            _overlap["wgrad"] += 1
            self._home = _overlap["home"]
        return self

    def __exit__(self, *exc):
        with _overlap_lock:
            _overlap["wgrad"] -= 1
            if _overlap["wgrad"] == 0:
                _overlap["home"] = None
        home = self._home
        if home is not None and _here(home[0]) != home:
            torch.cuda.current_stream(home[0]).wait_stream(_stream(home))
        K.join_side_streams(since=self._mark)
        return False


# A weight gradient below this many FLOPs stays on the data-gradient chain's
# stream, where that is the context's (a product in line on another stream
# would need waits of its own to stay ordered): the two cross-stream waits of
# the side stream take the host 30-40 us and the GPU 8-12 us, as long as such a
# product runs (8.6 GFLOP: 18 us).
_SIDE_MIN_FLOPS = 1.2e10


def _fp32_accum_target(param):
    """(main_grad, accumulate): the fp32 buffer the kernel writes param's
    gradient into, and whether it adds (False for the first contribution
    after a deferred zero_grad_buffer(), when it stores).  (None, False) when
    param has no fp32 main_grad: the gradient is then returned."""
    mg = getattr(param, "main_grad", None)
    if mg is None or mg.dtype != torch.float32:
        return None, False
    return main_grad_target(param)


def _pair_target(p1, p2):
    """(main_grad 1, main_grad 2, accumulate) for two gradients one kernel
    call writes under one accumulate flag (LayerNorm gamma and beta).  If
    only one of them is stale, that one is zeroed now and both accumulate;
    (None, None, False) unless both have a main_grad (stale flags are then
    left as they were)."""
    for p in (p1, p2):
        mg = getattr(p, "main_grad", None)
        if mg is None or mg.dtype != torch.float32:
            return None, None, False
    s1 = getattr(p1, "_eth_main_grad_stale", False)
    s2 = getattr(p2, "_eth_main_grad_stale", False)
    if s1 and s2:
        p1._eth_main_grad_stale = p2._eth_main_grad_stale = False
        return p1.main_grad, p2.main_grad, False
    return materialize_main_grad(p1), materialize_main_grad(p2), True


def _flat(x):
    return x if x.dim() == 2 else x.reshape(-1, x.shape[-1])


def _wgrad(weight, dy2, x2, mg, accumulate):
    """weight's gradient into its fp32 main grad: inside overlapped_wgrad on a
    side stream, or in line when it is small and the node runs on the
    context's own stream.  `weight._eth_side_grad` says which of the two the
    last contribution took; each waits for the other, so contributions to a
    weight form one chain."""
    if not _overlap["wgrad"] or not dy2.is_cuda:
        K.gemm(dy2.t(), x2, out=mg, accumulate=accumulate)
        return
    device, home = dy2.device, _overlap["home"]
    here = _here(device.index)
    if here == home and 2.0 * dy2.numel() * x2.shape[1] < _SIDE_MIN_FLOPS:
        if getattr(weight, "_eth_side_grad", False):
            torch.cuda.current_stream(device).wait_stream(K.side_stream(device))
        weight._eth_side_grad = False
        K.gemm(dy2.t(), x2, out=mg, accumulate=accumulate)
        return
    # the weight gradient only feeds main_grad: it runs on a side stream,
    # overlapped with the data-gradient chain, and is joined before the
    # gradient sync reads the buffer
    side = K.side_stream(device)
    K.mark_side_launch()
    side.wait_stream(torch.cuda.current_stream(device))
    if here != home and home is not None and not getattr(weight, "_eth_side_grad", True):
        side.wait_stream(_stream(home))
    weight._eth_side_grad = True
    with torch.cuda.stream(side):
        K.gemm(dy2.t(), x2, out=mg, accumulate=accumulate)
    dy2.record_stream(side)
    x2.record_stream(side)


def _chained(weight, device):
    """Orders a contribution to weight's main grad on the current stream into the
    chain that _wgrad forms: waits for the last one, and returns what is called
    behind the new one."""
    if not _overlap["wgrad"]:
        return lambda: None
    home, here = _overlap["home"], _here(device.index)
    side, current = K.side_stream(device), torch.cuda.current_stream(device)
    last = getattr(weight, "_eth_side_grad", None)
    if last:
        current.wait_stream(side)
    elif last is False and home is not None and here != home:
        current.wait_stream(_stream(home))

    def after():
        weight._eth_side_grad = here != home
        if here != home:
            K.mark_side_launch()
            side.wait_stream(current)

    return after


class LinearFn(torch.autograd.Function):
    """y = x @ W^T (+ b): ColumnParallelLinear / RowParallelLinear at TP=1."""

    @staticmethod
    def forward(ctx, x, weight, bias):
        x2 = _flat(x.contiguous())
        y = K.gemm(x2, weight.t(), bias=bias)
        ctx.save_for_backward(x2, weight, bias)
        ctx.in_shape = x.shape
        return y.view(*x.shape[:-1], weight.shape[0])

    @staticmethod
    def backward(ctx, dy):
        x2, weight, bias = ctx.saved_tensors
        dy2 = _flat(dy.contiguous())
        dx = K.gemm(dy2, weight).view(ctx.in_shape) if ctx.needs_input_grad[0] else None
        dw = db = None
        if ctx.needs_input_grad[1]:
            mg, accumulate = _fp32_accum_target(weight)
            if mg is not None:
                _wgrad(weight, dy2, x2, mg, accumulate)
                grad_written(weight)
            else:
                # one rounding of the fp32 product to the parameter dtype
                dw = K.gemm(dy2.t(), x2, out_dtype=weight.dtype)
        if bias is not None and ctx.needs_input_grad[2]:
            mg, accumulate = _fp32_accum_target(bias)
            if mg is not None:
                K.col_sum(dy2, mg, accumulate=accumulate)
                grad_written(bias)
            else:
                acc = torch.empty(bias.shape, dtype=torch.float32, device=bias.device)
                K.col_sum(dy2, acc, accumulate=False)
                db = acc.to(bias.dtype)
        return dx, dw, db


class LayerNormFn(torch.autograd.Function):
    """MixedFusedLayerNorm (model/fused_layer_norm.py:30-89)."""

    @staticmethod
    def forward(ctx, x, gamma, beta, eps):
        xc = x.contiguous()
        y, mean, rstd = K.layer_norm_fwd(_flat(xc), gamma, beta, eps)
        ctx.save_for_backward(xc, gamma, beta, mean, rstd)
        return y.view(x.shape)

    @staticmethod
    def backward(ctx, dy):
        x, gamma, beta, mean, rstd = ctx.saved_tensors
        dg, db, acc = _pair_target(gamma, beta)
        own = dg is None
        if own:
            dg = torch.empty(gamma.shape, dtype=torch.float32, device=x.device)
            db = torch.empty(beta.shape, dtype=torch.float32, device=x.device)
        dx = K.layer_norm_bwd(_flat(dy.contiguous()), _flat(x), mean, rstd, gamma, dg, db, accumulate=acc)
        if not own:
            grad_written(gamma)
            grad_written(beta)
            return dx.view(x.shape), None, None, None
        return dx.view(x.shape), dg.to(gamma.dtype), db.to(beta.dtype), None


class TransposedLayerNormFn(torch.autograd.Function):
    """The final LayerNorm of the GPT stage, x.transpose(0, 1).contiguous()
    then MixedFusedLayerNorm (flex_ops.py final-layernorm, :552-553): [s, b, h]
    in, [b, s, h] out, with the row permutation done by the LayerNorm
    kernels' own reads and writes instead of two transposing copies."""

    @staticmethod
    def forward(ctx, x, gamma, beta, eps):
        xc = x.contiguous()
        y, mean, rstd = K.layer_norm_fwd_sb(xc, gamma, beta, eps)
        ctx.save_for_backward(xc, gamma, beta, mean, rstd)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, gamma, beta, mean, rstd = ctx.saved_tensors
        dg, db, acc = _pair_target(gamma, beta)
        own = dg is None
        if own:
            dg = torch.empty(gamma.shape, dtype=torch.float32, device=x.device)
            db = torch.empty(beta.shape, dtype=torch.float32, device=x.device)
        dx = K.layer_norm_bwd_sb(dy.contiguous(), x, mean, rstd, gamma, dg, db, accumulate=acc)
        if not own:
            grad_written(gamma)
            grad_written(beta)
            return dx, None, None, None
        return dx, dg.to(gamma.dtype), db.to(beta.dtype), None


class LayerNormResidualFn(torch.autograd.Function):
    """MixedFusedLayerNorm whose input also feeds a later residual add:
    returns (LayerNorm(x), x).  The second output is what the op publishes
    as the residual (hidden_states_1/2, flex_ops.py:488-664), so both
    gradients of x arrive in one backward call and are added inside the
    LayerNorm backward kernel instead of by autograd's accumulation.  When x
    was produced by an op (not a leaf), the backward also leaves the
    column-sum partials of the returned gradient on it as
    `_eth_colsum_part`: BiasDropoutAddFn's backward folds them into its bias
    gradient instead of summing that gradient again."""

    @staticmethod
    def forward(ctx, x, gamma, beta, eps):
        ctx.set_materialize_grads(False)
        xc = x.contiguous()
        pre = getattr(x, "_eth_ln_fwd", None)
        if pre is not None:
            # the bias-dropout-add that made x already normalized it for this
            # LayerNorm (BiasDropoutAddLayerNormFn): taken once
            del x._eth_ln_fwd
        if pre is not None and pre[0] is gamma and pre[1] is beta and pre[2] == eps:
            y, mean, rstd = pre[3], pre[4], pre[5]
        else:
            y, mean, rstd = K.layer_norm_fwd(_flat(xc), gamma, beta, eps)
        ctx.save_for_backward(xc, gamma, beta, mean, rstd)
        ctx.colsum = x.grad_fn is not None
        return y.view(x.shape), x.view_as(x)

    @staticmethod
    def backward(ctx, dy, dres):
        x, gamma, beta, mean, rstd = ctx.saved_tensors
        if dy is None:
            return dres, None, None, None
        dg, db, acc = _pair_target(gamma, beta)
        own = dg is None
        if own:
            dg = torch.empty(gamma.shape, dtype=torch.float32, device=x.device)
            db = torch.empty(beta.shape, dtype=torch.float32, device=x.device)
        part = None
        if dres is None:
            dx = K.layer_norm_bwd(_flat(dy.contiguous()), _flat(x), mean, rstd, gamma, dg, db, accumulate=acc)
        else:
            out = K.layer_norm_bwd(_flat(dy.contiguous()), _flat(x), mean, rstd, gamma, dg, db, accumulate=acc,
                                   dresid=_flat(dres.contiguous()), colsum=ctx.colsum)
            dx, part = out if ctx.colsum else (out, None)
        dx = dx.view(x.shape)
        if part is not None:
            dx._eth_colsum_part = part
        if not own:
            grad_written(gamma)
            grad_written(beta)
            return dx, None, None, None
        return dx, dg.to(gamma.dtype), db.to(beta.dtype), None


def _whole(t):
    """t contiguous and 16-byte aligned (its own memory where it is)."""
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


class GatedResidualNormFn(torch.autograd.Function):
    """(h, y): h = residual_scale * residual + gate * norm(x), the residual
    stream behind a block whose output x is normed (post_gamma, post_beta) and
    gated (gate [cols], None: one), and y = norm(h) (gamma, beta) for the next
    block, in one pass.  The norms are LayerNorms, or with `rms` root-mean-square
    norms without betas (None)."""

    @staticmethod
    def forward(ctx, x, residual, post_gamma, post_beta, gate, residual_scale, gamma, beta, eps=1e-5, rms=False):
        ctx.set_materialize_grads(False)
        if residual.shape != x.shape:
            raise ValueError(f"residual {tuple(residual.shape)} does not match x {tuple(x.shape)}")
        xc, rc, scale = _whole(x), _whole(residual), float(residual_scale)
        h, y, stats = K.residual_norm_fwd(xc, rc, post_gamma, post_beta, gate, scale, gamma, beta, eps, rms)
        ctx.save_for_backward(xc, rc, stats, post_gamma, post_beta, gate, gamma, beta)
        ctx.scale, ctx.eps, ctx.rms = scale, eps, rms
        return h, y

    @staticmethod
    def backward(ctx, dh, dy):
        if dh is None and dy is None:
            return (None,) * 10
        x, residual, stats, *params = ctx.saved_tensors
        needs = ctx.needs_input_grad
        wanted = needs[2], needs[3], needs[4], needs[6], needs[7]
        # gradients that are returned share one allocation
        new = iter(torch.empty(sum(wanted), x.shape[-1], dtype=x.dtype, device=x.device).unbind(0))
        targets, returned, places, added = [], [], set(), []
        for p, need in zip(params, wanted):
            target = result = None
            if need:
                mg, accumulate = _fp32_accum_target(p)
                if mg is None:
                    result = next(new)
                    target = result, False
                elif mg.data_ptr() in places:
                    # (one parameter in two places of the call: its second gradient is added behind it)
                    target = torch.empty(p.shape, dtype=torch.float32, device=p.device), False
                    added.append((mg, target[0]))
                else:
                    target = mg, accumulate
                    places.add(mg.data_ptr())
            targets.append(target)
            returned.append(result)
        pg, pb, gate, gamma, beta = params
        dx, dres = K.residual_norm_bwd(_whole(x), _whole(residual), stats, None if dh is None else _whole(dh),
                                       None if dy is None else _whole(dy), pg, pb, gate, ctx.scale, gamma, beta, ctx.eps,
                                       ctx.rms, targets, needs[0], needs[1])
        for mg, extra in added:
            mg.view(-1).add_(extra.view(-1))
        for p, t, r in zip(params, targets, returned):
            if t is not None and r is None:
                grad_written(p)
        dpg, dpb, dgate, dg, db = returned
        return dx, dres, dpg, dpb, dgate, None, dg, db, None, None


class BiasGeluFn(torch.autograd.Function):
    """gelu_tanh(x + b) (flex_ops.py:1882-1906)."""

    @staticmethod
    def forward(ctx, x, bias):
        xc = x.contiguous()
        y = K.bias_gelu_fwd(_flat(xc), bias)
        ctx.save_for_backward(xc, bias)
        return y.view(x.shape)

    @staticmethod
    def backward(ctx, dy):
        x, bias = ctx.saved_tensors
        db = None
        if ctx.needs_input_grad[1]:
            # the bias gradient (column sums of dx) comes out of the same pass
            mg, accumulate = _fp32_accum_target(bias)
            target = mg if mg is not None else torch.empty(bias.shape, dtype=torch.float32, device=bias.device)
            dx = K.bias_gelu_bwd(_flat(dy.contiguous()), _flat(x), bias, dbias=target, accumulate=accumulate)
            if mg is None:
                db = target.to(bias.dtype)
            else:
                grad_written(bias)
        else:
            dx = K.bias_gelu_bwd(_flat(dy.contiguous()), _flat(x), bias)
        return dx.view(x.shape), db


class BiasDropoutAddFn(torch.autograd.Function):
    """residual + dropout(x + b, p) (flex_ops.py:104-134)."""

    @staticmethod
    def forward(ctx, x, bias, residual, p, seed):
        out = K.bias_dropout_add_fwd(_flat(x.contiguous()), bias, _flat(residual.contiguous()), p=p, seed=seed)
        ctx.p, ctx.seed = p, seed
        ctx.save_for_backward(bias)
        return out.view(x.shape)

    @staticmethod
    def backward(ctx, dout):
        return _bias_dropout_add_bwd(ctx, dout)


class BiasDropoutAddLayerNormFn(torch.autograd.Function):
    """BiasDropoutAddFn whose output the next op normalizes with `ln` (its
    LayerNorm module): one kernel also produces that LayerNorm's output,
    mean and rstd, returned as non-differentiable outputs for
    LayerNormResidualFn to take over, so the LayerNorm does not read h back.
    Gradients are BiasDropoutAddFn's; the LayerNorm keeps its own node."""

    @staticmethod
    def forward(ctx, x, bias, residual, p, seed, ln):
        # no zero tensors for the gradients of y, mean, rstd: they have none
        ctx.set_materialize_grads(False)
        h, y, mean, rstd = K.bias_dropout_add_layer_norm_fwd(
            _flat(x.contiguous()), bias, _flat(residual.contiguous()), ln.weight, ln.bias, p=p, seed=seed,
            eps=ln.eps)
        ctx.p, ctx.seed = p, seed
        ctx.save_for_backward(bias)
        ctx.mark_non_differentiable(y, mean, rstd)
        return h.view(x.shape), y.view(x.shape), mean, rstd

    @staticmethod
    def backward(ctx, dout, _dy, _dmean, _drstd):
        if dout is None:
            return None, None, None, None, None, None
        return (*_bias_dropout_add_bwd(ctx, dout), None)


def _bias_dropout_add_bwd(ctx, dout):
    """Gradients of residual + dropout(x + b) for (x, bias, residual, p, seed)."""
    (bias,) = ctx.saved_tensors
    part = getattr(dout, "_eth_colsum_part", None) if ctx.p == 0 else None
    dout = dout.contiguous()
    dx = K.dropout_bwd(_flat(dout), ctx.p, ctx.seed).view(dout.shape) if ctx.p > 0 else dout
    db = None
    if ctx.needs_input_grad[1]:
        mg, accumulate = _fp32_accum_target(bias)
        target = mg if mg is not None else torch.empty(bias.shape, dtype=torch.float32, device=bias.device)
        if part is not None:
            # column sums already produced by the LayerNorm backward that
            # made dout (p == 0: dx is dout)
            K.reduce_partials(part, target, accumulate=accumulate)
        else:
            K.col_sum(_flat(dx), target, accumulate=accumulate)
        if mg is None:
            db = target.to(bias.dtype)
        else:
            grad_written(bias)
    return dx, db, dout, None, None


class SplitQKVFn(torch.autograd.Function):
    """[s, b, np, 3*hn] -> q, k, v views (split_tensor_along_last_dim,
    mpu/utils.py:33-52) without copies.  When the incoming gradients are the
    three views of one [s, b, np, 3*hn] buffer (what attention's backward
    writes), that buffer is passed back as is."""

    @staticmethod
    def forward(ctx, mixed, hn):
        ctx.hn = hn
        ctx.shape = mixed.shape
        q, k, v = torch.split(mixed, hn, dim=-1)
        return q, k, v

    @staticmethod
    def backward(ctx, dq, dk, dv):
        hn = ctx.hn
        base = getattr(dq, "_eth_qkv_base", None)
        if base is not None and dk is not None and dv is not None:
            return base, None
        out = torch.zeros(ctx.shape, dtype=(dq if dq is not None else dk).dtype, device=(dq if dq is not None else dk).device)
        for i, g in enumerate((dq, dk, dv)):
            if g is not None:
                out[..., i * hn : (i + 1) * hn].copy_(g)
        return out, None


class CausalAttentionFn(torch.autograd.Function):
    """softmax(QK^T/sqrt(hn) + causal) V on [s, b, np, hn] views -> [s, b, np*hn]."""

    @staticmethod
    def forward(ctx, q, k, v):
        out, lse = K.attention_fwd(q, k, v)
        ctx.save_for_backward(q, k, v, out, lse)
        return out

    @staticmethod
    def backward(ctx, dout):
        q, k, v, out, lse = ctx.saved_tensors
        s, b, n, hn = q.shape
        dqkv = torch.empty(s, b, n, 3 * hn, dtype=q.dtype, device=q.device)
        dq, dk, dv = torch.split(dqkv, hn, dim=-1)
        K.attention_bwd(q, k, v, out, dout.contiguous(), lse, dq, dk, dv)
        dq._eth_qkv_base = dqkv
        return dq, dk, dv


class PackedCausalAttentionFn(torch.autograd.Function):
    """softmax(scale QK^T + causal) V within each sequence of `packed`
    (eth_amd.packed.PackedSequences) on q [rows, n, hn] and k, v [rows, m, hn]
    views -> [rows, n*hn]; n / m query heads share each key and value head.
    Rows of no sequence give zeros and get zero gradients.  scale: 1/sqrt(hn)
    unless given.  A value that is not finite reaches the outputs of its own
    sequence only, of the rows behind it and of those before it in the same
    64-row block (a product of a masked zero with it is NaN); gradients of any
    row of the sequence."""

    @staticmethod
    def forward(ctx, q, k, v, packed, scale=None):
        scale = None if scale is None else float(scale)  # (a tensor's value of now)
        out, lse = K.packed_attention_fwd(q, k, v, packed, scale)
        ctx.packed, ctx.scale = packed, scale
        ctx.save_for_backward(q, k, v, out, lse)
        return out

    @staticmethod
    def backward(ctx, dout):
        q, k, v, out, lse = ctx.saved_tensors
        return (*K._packed_attention_grads(q, k, v, out, dout, lse, ctx.packed, ctx.scale), None, None)


class EmbeddingFn(torch.autograd.Function):
    """word[tokens] + pos[positions] -> [s, b, h] (Embedding_v1, dropout p = 0
    handled by the caller)."""

    @staticmethod
    def forward(ctx, word, pos, tokens, positions, bad_flag):
        out = K.embedding_fwd(tokens, positions, word, pos, bad_flag)
        ctx.save_for_backward(tokens, positions, word, pos)
        return out

    @staticmethod
    def backward(ctx, dout):
        tokens, positions, word, pos = ctx.saved_tensors
        # the scatter-add needs real values underneath: stale buffers are
        # zeroed first; 16-bit main grads receive the returned gradient
        # through the DDP hook
        def fp32_target(p):
            mg = getattr(p, "main_grad", None)
            return materialize_main_grad(p) if mg is not None and mg.dtype == torch.float32 else None

        mw, mp = fp32_target(word), fp32_target(pos)
        gw = mw if mw is not None else torch.zeros(word.shape, dtype=torch.float32, device=word.device)
        gp = mp if mp is not None else torch.zeros(pos.shape, dtype=torch.float32, device=pos.device)
        K.embedding_bwd(tokens, positions, dout.contiguous(), gw, gp)
        for p, m in ((word, mw), (pos, mp)):
            if m is not None:
                grad_written(p)
        return (None if mw is not None else gw.to(word.dtype), None if mp is not None else gp.to(pos.dtype), None,
                None, None)


class CrossEntropyFn(torch.autograd.Function):
    """Per-token loss of 16-bit logits [..., V] against int64 labels [...]
    (vocab_parallel_cross_entropy at TP = 1, computed in fp32)."""

    @staticmethod
    def forward(ctx, logits, labels, bad_flag):
        shape = logits.shape[:-1]
        z = logits.reshape(-1, logits.shape[-1])
        lab = labels.reshape(-1).contiguous()
        loss, lse = K.xent_fwd(z, lab, bad_flag)
        ctx.save_for_backward(z, lab, lse)
        ctx.shape = logits.shape
        return loss.view(shape)

    @staticmethod
    def backward(ctx, dloss):
        z, lab, lse = ctx.saved_tensors
        dz = K.xent_bwd(z, lab, lse, dloss.reshape(-1).float().contiguous())
        return dz.view(ctx.shape), None, None


def _logit_rows(logits):
    """[rows, V] of logits [..., V] for the row kernels: the tensor's own
    memory where its rows are whole and apart, else a copy."""
    z = logits if logits.dim() == 2 else logits.reshape(-1, logits.shape[-1])
    rows, V = z.shape
    s0, s1 = z.stride()
    return z if (V == 1 or s1 == 1) and (rows <= 1 or s0 >= V) else z.contiguous()


def _row_values(t):
    """An upstream gradient of row values as contiguous fp32, in any shape
    (autograd gives it the values' own shape and device)."""
    if t is None or t.dtype == torch.float32 and t.is_contiguous():
        return t
    return t.float().contiguous()


class TokenLogprobsFn(torch.autograd.Function):
    """Log probabilities of tokens [...] under logits [..., V] (bf16, fp16 or
    fp32), the entropy of each row and its top_k largest log probabilities with
    their ids: (logprob [...], entropy [...], top_logprobs [..., top_k],
    top_ids [..., top_k]).  Gradients flow from logprob and entropy; the top
    alternatives are values.  Rows whose token is `ignore_index` give 0, 0,
    -inf and -1 and get no gradient."""

    @staticmethod
    def forward(ctx, logits, tokens, top_k, bad_flag, ignore_index=-100):
        ctx.set_materialize_grads(False)
        shape = tokens.shape
        if shape != logits.shape[:-1]:
            raise ValueError(f"tokens {tuple(shape)} do not match logits {tuple(logits.shape)}")
        z, t = _logit_rows(logits), tokens.reshape(-1).contiguous()
        logprob, entropy, stats, top, ids, ctx.layout = K._token_logprobs_fwd(z, t, top_k, bad_flag, ignore_index, shape)
        ctx.save_for_backward(z, t, stats, entropy)
        ctx.shape, ctx.ignore_index = logits.shape, ignore_index
        ctx.mark_non_differentiable(top, ids)
        return logprob, entropy, top, ids

    @staticmethod
    def backward(ctx, dlogprob, dentropy, _dtop, _dids):
        if dlogprob is None and dentropy is None:
            return None, None, None, None, None
        z, t, stats, entropy = ctx.saved_tensors
        f32 = torch.float32
        layout = K._saved_layout(ctx.layout, z, (t, torch.int64), (stats, f32), (entropy, f32))
        dz = K._token_logprobs_bwd(layout, z, t, stats, entropy, _row_values(dlogprob), _row_values(dentropy),
                                   ctx.ignore_index, ctx.shape)
        return dz, None, None, None, None


class TopkDistillFn(torch.autograd.Function):
    """Per-row distillation loss [...] of logits [..., V] on a teacher's top
    logits teacher_logits [..., k] at teacher_ids [..., k] (int64; negative: no
    entry): temperature^2 KL(q || p) with q over the row's entries and p over
    the vocabulary, both at the temperature.  The teacher is a constant."""

    @staticmethod
    def forward(ctx, logits, teacher_ids, teacher_logits, temperature, bad_flag):
        shape, temperature = logits.shape[:-1], float(temperature)
        if teacher_ids.shape[:-1] != shape or teacher_logits.shape != teacher_ids.shape:
            raise ValueError(f"teacher ids {tuple(teacher_ids.shape)} and logits {tuple(teacher_logits.shape)} do not "
                             f"match logits {tuple(logits.shape)}")
        z = _logit_rows(logits)
        if len(shape) != 1:
            teacher_ids, teacher_logits = (t.reshape(z.shape[0], t.shape[-1]) for t in (teacher_ids, teacher_logits))
        ids, teacher = teacher_ids.contiguous(), teacher_logits.contiguous()
        loss, stats, ctx.layout = K._topk_distill_fwd(z, ids, teacher, temperature, bad_flag, shape)
        ctx.save_for_backward(z, ids, teacher, stats)
        ctx.shape, ctx.temperature, ctx.bad_flag, ctx.teacher = logits.shape, temperature, bad_flag, teacher.dtype
        return loss

    @staticmethod
    def backward(ctx, dloss):
        z, ids, teacher, stats = ctx.saved_tensors
        layout = K._saved_layout(ctx.layout, z, (ids, torch.int64), (teacher, ctx.teacher), (stats, torch.float32))
        dz = K._topk_distill_bwd(layout, z, ids, teacher, ctx.temperature, stats, _row_values(dloss), ctx.bad_flag,
                                 ctx.shape)
        return dz, None, None, None, None


def _aligned_rows(x):
    """x [..., H] as [rows, H] whose rows the kernels can read in place: its own
    memory where they are whole, apart and 16-byte aligned, else a copy."""
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    rows, cols = x2.shape
    s0, s1 = x2.stride()
    if (cols > 1 and s1 != 1) or (rows > 1 and (s0 < cols or s0 % 8)):
        return x2.clone(memory_format=torch.contiguous_format)
    return x2.clone() if x2.data_ptr() % 16 else x2


def _aligned_target(mg, accumulate):
    """(tensor for the kernel, whether it adds, what is called behind it) for a main
    grad that may start anywhere in its buffer: itself where it is 16-byte aligned,
    else a tensor that is stored or added there."""
    if mg.data_ptr() % 16 == 0:
        return mg, accumulate, lambda: None
    own = torch.empty_like(mg)
    return own, False, lambda: mg.add_(own) if accumulate else mg.copy_(own)


class LinearCrossEntropyFn(torch.autograd.Function):
    """Per-token loss [...] (fp32) of the head's logits hidden [..., H] @
    weight[V, H]^T against int64 labels [...]: LinearFn and CrossEntropyFn in
    one, without the logits in memory.  Rows whose label is `ignore_index` have
    loss 0, are not read and get no gradient."""

    @staticmethod
    def forward(ctx, hidden, weight, labels, bad_flag, ignore_index=-100):
        if labels.shape != hidden.shape[:-1]:
            raise ValueError(f"labels {tuple(labels.shape)} do not match hidden {tuple(hidden.shape)}")
        h, lab = _aligned_rows(hidden), labels.reshape(-1).contiguous()
        loss, lse = K.linear_xent_fwd(h, weight, lab, bad_flag, ignore_index)
        ctx.save_for_backward(h, weight, lab, lse)
        ctx.shape, ctx.ignore_index = hidden.shape, ignore_index
        return loss.view(labels.shape)

    @staticmethod
    def backward(ctx, dloss):
        h, weight, lab, lse = ctx.saved_tensors
        need_h, need_w = ctx.needs_input_grad[:2]
        mg, accumulate = _fp32_accum_target(weight) if need_w else (None, False)
        target = mg
        if mg is not None:
            after = _chained(weight, h.device)
            target, accumulate, settle = _aligned_target(mg, accumulate)
        dh, dw = K.linear_xent_bwd(_aligned_rows(h), weight, lab, lse, _row_values(dloss.reshape(-1)), ctx.ignore_index,
                                   need_h, need_w, target, accumulate)
        if mg is not None:
            settle()
            after()
            grad_written(weight)
            dw = None
        return None if dh is None else dh.view(ctx.shape), dw, None, None, None


def _adapter_targets(params, needs):
    """[(pair for K.adapter_linear_bwd, gradient to return, what is called behind
    it)] of lora_a and lora_b."""
    targets, places = [], set()
    for p, need in zip(params, needs):
        mg, accumulate = _fp32_accum_target(p) if need else (None, False)
        if not need:
            targets.append((None, None, lambda: None))
        elif mg is None:
            new = torch.empty(p.shape, dtype=p.dtype, device=p.device)
            targets.append(((new, False), new, lambda: None))
        elif mg.data_ptr() in places:
            # (one parameter in both places: its second gradient is added behind the first)
            new = torch.empty(p.shape, dtype=torch.float32, device=p.device)
            targets.append(((new, False), None, lambda mg=mg, new=new: mg.add_(new)))
        else:
            places.add(mg.data_ptr())
            target, accumulate, settle = _aligned_target(mg, accumulate)
            targets.append(((target, accumulate), None, settle))
    return targets


class AdapterLinearFn(torch.autograd.Function):
    """y = x @ W^T (+ bias) + scale (x @ A^T) @ B^T: LinearFn with each row's
    low-rank adapter beside the shared weight; A [r, in] and B [out, r] of lora_a
    [adapters, r, in] and lora_b [adapters, out, r], adapters and scales of the rows
    by `rows` (eth_amd.packed.AdapterRows, whose total are x's rows).  Rows of no
    adapter are LinearFn's."""

    @staticmethod
    def forward(ctx, x, weight, bias, lora_a, lora_b, rows):
        x2 = _aligned_rows(x)
        y, saved = K.adapter_linear_fwd(x2, weight, bias, lora_a, lora_b, rows, save=ctx.needs_input_grad[4])
        ctx.save_for_backward(x2, weight, bias, lora_a, lora_b, *(saved or ()))
        ctx.rows, ctx.in_shape = rows, x.shape
        return y.view(*x.shape[:-1], weight.shape[0])

    @staticmethod
    def backward(ctx, dy):
        x2, weight, bias, lora_a, lora_b, *saved = ctx.saved_tensors
        x2, dy2 = _aligned_rows(x2), _whole(dy).view(-1, weight.shape[0])
        needs = ctx.needs_input_grad
        (da, ga, settle_a), (db, gb, settle_b) = _adapter_targets((lora_a, lora_b), needs[3:5])
        dx = K.adapter_linear_bwd(x2, weight, lora_a, lora_b, dy2, ctx.rows, tuple(t.contiguous() for t in saved) or None,
                                  needs[0], da, db)
        settle_a()
        settle_b()
        for p, pair, g in ((lora_a, da, ga), (lora_b, db, gb)):
            if pair is not None and g is None:
                grad_written(p)
        dw = dbias = None
        if needs[1]:
            mg, accumulate = _fp32_accum_target(weight)
            pad = -x2.shape[0] % 8  # (the product takes depths that are multiples of 8)
            dyw, xw = (torch.nn.functional.pad(t, (0, 0, 0, pad)) if pad else t for t in (dy2, x2))
            if mg is not None:
                _wgrad(weight, dyw, xw, mg, accumulate)
                grad_written(weight)
            else:
                dw = K.gemm(dyw.t(), xw, out_dtype=weight.dtype)
        if bias is not None and needs[2]:
            mg, accumulate = _fp32_accum_target(bias)
            acc = mg if mg is not None else torch.empty(bias.shape, dtype=torch.float32, device=bias.device)
            K.col_sum(dy2, acc, accumulate=accumulate)
            if mg is None:
                dbias = acc.to(bias.dtype)
            else:
                grad_written(bias)
        return None if dx is None else dx.view(ctx.in_shape), dw, dbias, ga, gb, None
