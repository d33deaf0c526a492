"""A layer of routed experts for a few tokens (a decoded batch): two kernels that read every chosen expert's weights once."""
import torch

from ... import _native_ops
from ._tensors import CODE, E4M3, check, groups, matrix, on_gpu, stream_of

MAX_TOKENS = 64


def _experts(name, w, e, rows, cols, device):
    """[e, rows, cols] weights with contiguous rows; returns the strides from expert to expert and row to row."""
    if w.device != device or w.dim() != 3 or w.shape != (e, rows, cols):
        raise ValueError(f"{name} must have shape ({e}, {rows}, {cols}) on {device}, got {tuple(w.shape)} on {w.device}")
    s = w.stride()
    if s[2] != 1:
        raise ValueError(f"{name}: the elements of a row must lie side by side, got strides {s}")
    return s[0], s[1]


def _block_scales(name, s, w, device):
    want = (w.shape[0], groups(w.shape[1]), groups(w.shape[2]))
    if s is None or s.dtype is not torch.float32 or s.device != device or tuple(s.shape) != want or not s.is_contiguous():
        raise ValueError(f"{name} must be a contiguous torch.float32 tensor of shape {want} on {device}")
    return s.data_ptr()


def moe_layer(x, logits, topk, w13, w2, w13_scale=None, w2_scale=None, renormalize=True, out=None):
    """out[t] = sum over the experts e that token t chooses: p[t, e] * W2_e (silu(W1_e x_t) * (W3_e x_t)) -> (out, ids, probs).

    x            [T, H] bfloat16 or float16, T <= 64
    logits       [T, E] float32, the router's answer: the topk largest choose (equal ones: the lower expert), p is their
                 softmax (renormalize) or the softmax over all experts.  -inf takes an expert out: it weighs 0 and adds
                 nothing even if fewer than topk others are left; a row of -inf alone gives zeros
    w13          [E, 2 I, H]: W1 (gate) in the first I rows, W3 (up) in the others; w2 [E, H, I].  e4m3 with scales for
                 blocks of 128 x 128, w13_scale [E, ceil(2 I / 128), ceil(H / 128)] and w2_scale [E, ceil(H / 128), ceil(I / 128)],
                 or bfloat16 (x bfloat16 too); rows contiguous and on 16 bytes.  H and I are multiples of 16
    out          [T, H] of x's type (default: a new tensor)
    ids, probs   [T, topk] int32 and float32: the choice, by falling logit, and its weights
    Sums are held in float32, the activations between the two products in 16 significant bits.  Every output row depends on its
    own token alone and comes out the same on every run.  Runs on torch's current stream; the workspace is torch's, per call."""
    device = on_gpu("x", x)
    if x.dim() != 2 or logits.dim() != 2 or w13.dim() != 3:
        raise ValueError("x and logits must be matrices, w13 and w2 [experts, rows, columns]")
    (t, h), e, two_i = x.shape, logits.shape[1], w13.shape[1]
    topk = int(topk)
    if two_i % 2:
        raise ValueError(f"w13 holds two weights of the same number of rows, got {two_i} rows")
    i = two_i // 2
    x_s = matrix("x", x, t, h, x.dtype, device)
    l_s = matrix("logits", logits, t, e, torch.float32, device)
    w13_e, w13_r = _experts("w13", w13, e, two_i, h, device)
    w2_e, w2_r = _experts("w2", w2, e, h, i, device)
    if w2.dtype is not w13.dtype or w13.dtype not in (E4M3, torch.bfloat16) or x.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"weights of {w13.dtype} and {w2.dtype} with x of {x.dtype}: e4m3 weights take bfloat16 or float16, bfloat16 weights bfloat16")
    s13 = s2 = 0
    if w13.dtype is E4M3:
        s13, s2 = _block_scales("w13_scale", w13_scale, w13, device), _block_scales("w2_scale", w2_scale, w2, device)
    elif w13_scale is not None or w2_scale is not None:
        raise ValueError("bfloat16 weights have no scales")
    need = _native_ops.moe_workspace_bytes(t, e, topk, h, i)
    if out is None:
        out = torch.empty((t, h), dtype=x.dtype, device=device)
    o_s = matrix("out", out, t, h, x.dtype, device)
    ids = torch.empty((t, topk), dtype=torch.int32, device=device)
    probs = torch.empty((t, topk), dtype=torch.float32, device=device)
    if t:
        ws = torch.empty(need, dtype=torch.uint8, device=device)
        check(_native_ops.lib().kcg_moe_layer(
            _native_ops.MOE_LAYER.pack(x.data_ptr(), logits.data_ptr(), w13.data_ptr(), s13, w2.data_ptr(), s2, out.data_ptr(), ids.data_ptr(),
                                       probs.data_ptr(), ws.data_ptr(), need, x_s, l_s, o_s, w13_e, w13_r, w2_e, w2_r, t, e, topk, h, i,
                                       CODE[x.dtype], CODE[w13.dtype], int(bool(renormalize))), device.index, stream_of(device.index)))
    return out, ids, probs
