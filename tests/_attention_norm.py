"""Attention over cached tokens held to a bound on the norm of its error.

Roundings of unit roundoff u that do not depend on each other are off by at most r = u / sqrt(3) in the root of their
mean square.  A result is off by r of its type for its own rounding, and for fp16 keys, values and weights by r of
2^-11 each: values and weights by r of the norm, keys by r sqrt(sum q^2 k^2 / sum of channels), which is 1.8 r for
queries N(0, 1) and keys N(0, 1) of which every 17th channel stands 6 higher.  fp16: r sqrt(3 + 1.8^2) = 7.0e-4; bf16:
sqrt(2.26e-3^2 + 6.4e-4^2) = 2.4e-3.  Kernels that keep the cache's codes exact are below that.  The bounds are those
figures and a third for what a norm over a hundred elements differs from its mean.

That takes many tokens with a say in a result.  Where a row's few largest weights decide, the error is that of their
logits, sum_j p_j e_j (v_j - o) with |e_j| <= 2^-11 scale sum |q k_j| for the keys' rounding; ``worst`` sums the
magnitudes of that, of 2^-11 of the weights (the same sum) and of the values, and of the result's own rounding.

A tile of 64 tokens that is lost among 9000 is 8e-2, one token 1e-2 and a mask off by one the same."""
import numpy as np
import torch

BOUND = {"f16": 1e-3, "bf16": 3e-3}


def definition(q, k, v, scale=None, weigh=None):
    """q [rows, heads, d], k and v [tokens, kv_heads, d], float64: the last row sees all tokens, the row before one fewer.
    ``weigh(p)`` changes the weights [heads, rows, tokens] that the oracle's own tests plant mistakes with."""
    q, k, v = (torch.as_tensor(x).double().cpu() for x in (q, k, v))
    rows, heads, d = q.shape
    tokens, kv_heads, _ = k.shape
    hide = torch.arange(tokens) > torch.arange(tokens - rows, tokens).view(-1, 1)
    out = torch.zeros_like(q)
    if tokens == 0:
        return out
    for h in range(kv_heads):
        at = slice(h * (heads // kv_heads), (h + 1) * (heads // kv_heads))
        z = (q[:, at].transpose(0, 1).flatten(0, 1) @ k[:, h].T).unflatten(0, (-1, rows))
        z = (z * (d ** -0.5 if scale is None else scale)).masked_fill(hide, -torch.inf)
        top = z.amax(-1, keepdim=True)
        p = torch.exp(z - torch.where(top == -torch.inf, 0.0, top))
        p = p if weigh is None else weigh(p)
        o = p.flatten(0, 1) @ v[:, h] / p.sum(-1).clamp_min(1e-300).view(-1, 1)
        out[:, at] = o.unflatten(0, (-1, rows)).transpose(0, 1)
    return out


def kept(x, group):
    """what the cache keeps of [tokens, heads, d], float64"""
    from test_attention_gpu import _params
    s, m = _params(x.float().cpu().numpy(), group)
    return torch.from_numpy(np.ascontiguousarray(s + m))


def close(got, want, dtype):
    """got within the bound of want [rows, heads, d], per head"""
    got, want = got.double().cpu(), want.double().cpu()
    err, size = (x.pow(2).sum((0, 2)).sqrt() for x in (got - want, want))
    return bool((err <= BOUND[dtype] * size + 1e-7).all())


def check(out, q, seqs, news, group, dtype, scale=None, first=0):
    """out and q [rows, heads, d]; sequence i has news[i] rows and the tokens seqs[i] = (k, v) [tokens, kv_heads, d]"""
    at = first
    for i, ((k, v), rows) in enumerate(zip(seqs, news)):
        if rows:
            want = definition(q[at:at + rows], kept(k, group), kept(v, v.shape[-1]), scale)
            assert close(out[at:at + rows], want, dtype), i
        at += rows


def worst(q, k, v, dtype, want):
    """the most that got - want can be to first order, by row and head, in the norm; and a tenth for higher orders"""
    q, k, v, want = (torch.as_tensor(x).double().cpu() for x in (q, k, v, want))
    (rows, heads, d), tokens, per = q.shape, len(k), q.shape[1] // k.shape[1]
    u = 2.0 ** -11
    hide = torch.arange(tokens) > torch.arange(tokens - rows, tokens).view(-1, 1)
    out = torch.zeros(rows, heads, dtype=torch.float64)
    for h in range(heads):
        kh, vh, o = k[:, h // per], v[:, h // per], want[:, h]
        p = torch.softmax((q[:, h] @ kh.T * d ** -0.5).masked_fill(hide, -torch.inf), -1)
        size = q[:, h].abs() @ kh.abs().T * d ** -0.5
        apart = (vh.pow(2).sum(-1) + o.pow(2).sum(-1, keepdim=True) - 2 * (o @ vh.T)).clamp_min(0).sqrt()
        own = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}[dtype] * o.pow(2).sum(-1).sqrt()
        out[:, h] = (p * (u * (1 + size) * apart + u * vh.pow(2).sum(-1).sqrt())).sum(-1) + own
    return 1.1 * out + 1e-7
