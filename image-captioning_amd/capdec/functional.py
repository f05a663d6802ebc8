"""Module-level compositions of the HIP ops used by the ``models`` classes.

Inference compositions call the forward kernels directly; training compositions (autograd enabled and
something requires grad) go through ``capdec.autograd`` Functions whose forward and backward are both
HIP kernels.  Nothing here falls back to ATen arithmetic.
"""
import torch

from . import ops


def _needs_graph(module, *tensors):
    return torch.is_grad_enabled() and (any(t.requires_grad for t in tensors) or
                                        any(p.requires_grad for p in module.parameters()))


def linear_dropout_bn(model, parts, x, dropout_first=False):
    """Feature head: for each (fc, lo, hi) in ``parts`` project x[:, lo:hi] with fc, concatenate the
    results column-wise, apply ``model.dropout`` (before the projection when ``dropout_first``) and
    ``model.batchnorm``.  Returns [B, len(parts)*E].

    eval: dropout is the identity and the BatchNorm (running statistics) is folded into the contraction's
    epilogue, so the head is one kernel per projection.  train: see ``capdec.autograd``.
    """
    bn = model.batchnorm
    if model.training:
        from . import autograd as AG
        return AG.head_train(model, parts, x, dropout_first)
    B = x.shape[0]
    E = parts[0][0].weight.shape[0]
    # a long contraction with few output tiles (the 86436-wide YOLO projection) is split over workgroups, its partial
    # sums added in a fixed order: the memory rows, and with them the decoded tokens, repeat exactly from run to run
    # (likewise a small batch in front of a 1000- or 2048-wide feature: at batch 32 the CNN head is four 64x64 tiles
    #  that each walk all 2048 k, 26.7 us on four of the chip's 256 compute units)
    few_tiles = ((B + 63) // 64) * ((E + 63) // 64) <= 32
    return ops.head_eval(x, [(fc.weight, fc.bias, lo, hi) for fc, lo, hi in parts], bn.weight, bn.bias,
                         bn.running_mean, bn.running_var, bn.eps,
                         lambda K: K >= 8192 or (few_tiles and K >= 1024))


def decoder_forward(dec, enc_output, captions, take_last=False):
    """Autograd-connected teacher-forced forward (reference transformer.py:125-138)."""
    from . import autograd as AG
    return AG.decoder_forward(dec, enc_output, captions, take_last)


def decoder_rnn_forward(rnn, features, captions):
    """``DecoderRNN.forward`` (reference cnnrnn_model.py:20-34): logits [B,T,V]."""
    if _needs_graph(rnn, features):
        from . import autograd as AG
        return AG.decoder_rnn_forward(rnn, features, captions)
    x0 = rnn.image_input(features)
    w = (rnn.lstm.weight_ih_l0, rnn.lstm.weight_hh_l0, rnn.lstm.bias_ih_l0, rnn.lstm.bias_hh_l0)
    h, c = ops.lstm_step(x0, None, None, *w)
    B, T = captions.shape
    emb = ops.embed_pe(captions, rnn.embed.weight, None).view(B, T, -1)
    Hd = h.shape[1]
    hs = torch.empty((B, T, Hd), device=h.device, dtype=torch.float32)
    for t in range(T):
        h, c = ops.lstm_step(emb[:, t], h, c, *w, h_out=hs[:, t])   # h' lands in the [B,T,Hd] slab
    return ops.linear(hs.view(B * T, Hd), rnn.fc2.weight, rnn.fc2.bias).view(B, T, -1)


def vocab_cross_entropy(x, weight, bias, targets, ignore_index=0, reduction="mean"):
    """Cross entropy of a vocabulary projection, ``cross_entropy(x @ weight.T + bias, targets)``, without the logits: they
    are formed tile by tile, in the forward pass and again, a piece of the vocabulary at a time, in the backward pass.

    x [..., K], weight [V, K] and bias [V] (or None) share one type: float32, bfloat16 or float16; targets [...] int64.
    Rows whose target is ``ignore_index`` have loss 0 and gradient 0 and are not read; any other target outside [0, V)
    makes the loss NaN.  reduction: "mean" over the counted rows (NaN if there are none; the gradients are zero then),
    "sum", or "none" (a loss per target).  The loss is float32; gradients flow to x, weight and bias in their own type.
    float32 operands above 64 rows are taken as pairs of float16 numbers scaled by the largest of each matrix (each row where
    nothing asks for a gradient): 22 bits, and steps of 2^-39 of that largest number.  They are multiplied as they are, which
    takes four to six times as long, where weight holds infinities and, if a gradient is asked for, where the largest numbers
    of two rows of x or of weight (zeros aside) are more than 2^16 apart.
    The gradient of the logits (a probability times a row's upstream gradient) is kept in the operands' own numbers: rounded
    to 16 bits for bfloat16 and float16, as a pair for float32 above 64 rows; in float16 and pairs what lies below 2^-38 of
    the largest upstream gradient is lost.

    There is no forward-mode derivative: an input that carries a tangent is refused.

    A backward pass that is to be captured in a HIP graph must not run while an eager graph of the same leaves is alive:
    drop the losses of earlier eager passes first."""
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"capdec: reduction must be 'mean', 'sum' or 'none', got {reduction!r}")
    if x.dim() < 1 or x.shape[:-1] != targets.shape:
        raise RuntimeError(f"capdec: x {tuple(x.shape)} and targets {tuple(targets.shape)} do not fit")
    x2, t = x.reshape(-1, x.shape[-1]), targets.reshape(-1)
    if (x2.stride(1) != 1 and x2.shape[1] > 1) or (x2.shape[0] > 1 and x2.stride(0) < x2.shape[1]):
        x2 = x2.contiguous()                       # columns apart, or rows that share memory (a broadcast x)
    t = t.contiguous()
    ins = (x2, weight) if bias is None else (x2, weight, bias)
    # (a tangent of forward-mode differentiation goes to the node as well, which refuses it rather than lose it)
    if x2.shape[0] == 0 or (torch.is_grad_enabled() and any(v.requires_grad for v in ins)) or \
            any(torch.autograd.forward_ad.unpack_dual(v).tangent is not None for v in ins):
        from . import autograd as AG
        loss = AG.vocab_cross_entropy(x2, weight, bias, t, ignore_index, reduction)
    else:
        nll, loss, _ = ops.vocab_ce_forward(x2, weight, bias, t, ignore_index, want_loss=reduction != "none", loss_only=True)
        loss = nll if reduction == "none" else loss[0 if reduction == "mean" else 1]
    return loss.view(targets.shape) if reduction == "none" else loss
