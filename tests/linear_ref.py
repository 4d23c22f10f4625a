"""Plain restatements, in 64 bits and token by token, of the linear half of a hybrid decoder: the short convolution of each
line's tokens, linear attention with decays (and the delta rule) over a state of each line, the gated norm and the join of a
block to its residual. Each also gives the size of what its results sum, which the tests' tolerances are multiples of."""
import torch


def conv(x, weight, state, cu, bias=None, silu=True):
    """(out, new state, size): size = sum |w x| + |bias|."""
    W, C = weight.shape[-1], x.shape[1]
    w = weight.double().reshape(C, W)
    out, size = torch.zeros(x.shape, dtype=torch.float64, device=x.device), torch.zeros_like(x, dtype=torch.float64)
    state = state.double().clone()
    for b in range(len(cu) - 1):
        rows = torch.cat((state[b], x[cu[b]:cu[b + 1]].double()))
        for i in range(cu[b + 1] - cu[b]):
            terms = rows[i:i + W].T * w
            y, s = terms.sum(1), terms.abs().sum(1)
            if bias is not None:
                y, s = y + bias.double(), s + bias.double().abs()
            out[cu[b] + i] = y / (1 + torch.exp(-y)) if silu else y
            size[cu[b] + i] = s
        state[b] = rows[len(rows) - (W - 1):]
    return out, state, size


def gates(decay, beta, a_log=None, dt_bias=None):
    """(log decay, beta) in 64 bits."""
    g, beta = decay.double(), None if beta is None else beta.double()
    if a_log is not None:
        g = g + (0 if dt_bias is None else dt_bias.double())
        g = -torch.exp(a_log.double()) * torch.logaddexp(g, torch.zeros_like(g))
        beta = None if beta is None else torch.sigmoid(beta)
    return torch.where(g > 0, torch.zeros_like(g), g), beta


def delta(q, k, v, decay, state, cu, beta=None, a_log=None, dt_bias=None, eps=1e-6, scale=None):
    """(out, new state, out size, state size): with W_t = exp(g) W_{t-1} + |u_t| |k_t| for each row of the state (W_0 its
    norm), which bounds the row's norm and every partial sum of it, the sizes are W_t |q_t| scale and W at the end."""
    T, Hk, Dk = q.shape
    Hv, Dv = v.shape[1:]
    scale = Dk ** -0.5 if scale is None else scale
    q, k, v = q.double(), k.double(), v.double()
    if eps is not None:
        q, k = (x / torch.sqrt(x.square().sum(-1, keepdim=True) + eps) for x in (q, k))
    q, k = (x.repeat_interleave(Hv // Hk, 1) for x in (q, k))
    g, beta = gates(decay, beta, a_log, dt_bias)
    out = torch.zeros((T, Hv, Dv), dtype=torch.float64, device=q.device)
    size = torch.zeros_like(out)
    S = state.double().clone()
    W = S.norm(dim=-1)
    for b in range(len(cu) - 1):
        for t in range(cu[b], cu[b + 1]):
            a = torch.exp(g[t])[:, None]
            S[b] *= a[..., None]
            u = v[t]
            if beta is not None:
                u = beta[t][:, None] * (u - torch.einsum("hvk,hk->hv", S[b], k[t]))
            S[b] += u[..., None] * k[t][:, None]
            W[b] = a * W[b] + u.abs() * k[t].norm(dim=-1, keepdim=True)
            out[t] = scale * torch.einsum("hvk,hk->hv", S[b], q[t])
            size[t] = scale * W[b] * q[t].norm(dim=-1, keepdim=True)
    return out, S, size, W


def rms(x, weight, eps, offset):
    return x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * (weight.double() + offset)


def gated(x, gate, weight, eps=1e-6, offset=0, activation="silu"):
    z = gate.double()
    s = 1 / (1 + torch.exp(-z))
    return rms(x.double(), weight, eps, offset) * (s * z if activation == "silu" else s)


def join(x, residual, weight, post=None, gate=None, scale=1.0, eps=1e-6, offset=0):
    """(sum, normed, size of the sum's terms)."""
    x = x.double()
    if post is not None:
        x = rms(x, post, eps, offset)
    if gate is not None:
        x = x * gate.double()
    total = residual.double() + scale * x
    return total, rms(total, weight, eps, offset), residual.double().abs() + (scale * x).abs()
