"""A layer of routed experts for a few tokens (a decoded batch): two kernels, or three, that read every chosen expert's weights once."""
from ... import _native_ops


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
    Sums are held in float32, the activations between the two products in 16 significant bits.  An output row is made of its
    own token alone and the same on every run (another number of tokens may cut its sums differently).  Runs on torch's current
    stream; the workspace is torch's, per call."""
    return _native_ops.torch_ops().moe_layer(x, logits, int(topk), w13, w2, w13_scale, w2_scale, renormalize, out)
