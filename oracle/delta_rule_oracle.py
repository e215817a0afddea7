"""float64 statement of the gated delta rule and of layer norm, token by token and row by row (test
infrastructure only).  Tensors may be on any device; everything is computed in float64."""
import torch


def _documents(B, T, lens):
    if lens is None:
        return [(b, 0, T) for b in range(B)]
    out, at = [], 0
    for n in lens:
        out.append((0, at, at + n))
        at += n
    return out


def delta_rule(q, k, v, g, beta, scale, state=None, lens=None, do=None, dstate=None):
    """o and the final state; with ``do`` also the gradients.  Returns a dict of float64 tensors.

    Forward per token: S <- e^g S; e = v - S^T k; u = beta e; S <- S + k u^T; o = scale S^T q.
    Backward per token, from the last: dS += scale q do^T; du = dS^T k; de = beta du;
    dk = dS u - Sd de; dSd = dS - k de^T; dg = <dSd, Sd>; dS <- e^g dSd (Sd: the decayed state)."""
    f = [t.detach().double() for t in (q, k, v, g, beta)]
    q, k, v, g, beta = f
    B, T, H, K = q.shape
    HV, V = v.shape[2:]
    rep = HV // H
    qh, kh = q.repeat_interleave(rep, 2), k.repeat_interleave(rep, 2)
    docs = _documents(B, T, lens)
    o = torch.zeros_like(v)
    finals, grads = [], {n: torch.zeros_like(t) for n, t in (('dq', qh), ('dk', kh), ('dv', v), ('dg', g), ('dbeta', beta))}
    dstates = []
    for n, (b, t0, t1) in enumerate(docs):
        S = state[n].detach().double() if state is not None else torch.zeros(HV, K, V, dtype=torch.float64, device=q.device)
        tape = []
        for t in range(t0, t1):
            Sd = torch.exp(g[b, t])[:, None, None] * S if not torch.isinf(g[b, t]).any() else torch.where(
                torch.isinf(g[b, t])[:, None, None], torch.zeros_like(S), torch.exp(g[b, t])[:, None, None] * S)
            e = v[b, t] - torch.einsum('hkv,hk->hv', Sd, kh[b, t])
            u = beta[b, t][:, None] * e
            S = Sd + kh[b, t][:, :, None] * u[:, None, :]
            o[b, t] = scale * torch.einsum('hkv,hk->hv', S, qh[b, t])
            tape.append((Sd, e, u, S))
        finals.append(S)
        if do is None:
            continue
        dS = dstate[n].detach().double() if dstate is not None else torch.zeros_like(S)
        for t in range(t1 - 1, t0 - 1, -1):
            Sd, e, u, S1 = tape.pop()
            d = do[b, t].detach().double()
            grads['dq'][b, t] = scale * torch.einsum('hkv,hv->hk', S1, d)
            dS = dS + scale * qh[b, t][:, :, None] * d[:, None, :]
            du = torch.einsum('hkv,hk->hv', dS, kh[b, t])
            de = beta[b, t][:, None] * du
            grads['dbeta'][b, t] = (du * e).sum(-1)
            grads['dv'][b, t] = de
            grads['dk'][b, t] = torch.einsum('hkv,hv->hk', dS, u) - torch.einsum('hkv,hv->hk', Sd, de)
            dS = dS - kh[b, t][:, :, None] * de[:, None, :]
            grads['dg'][b, t] = (dS * Sd).sum((-1, -2))
            dS = torch.where(torch.isinf(g[b, t])[:, None, None], torch.zeros_like(dS), torch.exp(g[b, t])[:, None, None] * dS)
        dstates.append(dS)
    out = {'o': o, 'state': torch.stack(finals)}
    if do is not None:
        for n in ('dq', 'dk'):
            grads[n] = grads[n].reshape(B, T, H, rep, K).sum(3)
        out.update(grads)
        out['dstate'] = torch.stack(dstates)
    return out


def norm(x, weight=None, bias=None, residual=None, gate=None, eps=1e-5, center=True, dy=None, dh=None):
    """y, h and, with ``dy``, the gradients, over rows of [R, D]."""
    d = lambda t: None if t is None else t.detach().double()  # noqa: E731
    x, weight, bias, residual, gate, dy, dh = (d(t) for t in (x, weight, bias, residual, gate, dy, dh))
    h = x if residual is None else x + residual
    D = h.shape[-1]
    mu = h.mean(-1, keepdim=True) if center else torch.zeros_like(h[..., :1])
    r = 1.0 / torch.sqrt(((h - mu) ** 2).mean(-1, keepdim=True) + eps)
    n = (h - mu) * r
    w = torch.ones(D, dtype=torch.float64, device=x.device) if weight is None else weight
    core = n * w + (0.0 if bias is None else bias)
    sg = None if gate is None else torch.sigmoid(gate)
    out = {'y': core if gate is None else core * gate * sg, 'h': h}
    if dy is None:
        return out
    dcore = dy if gate is None else dy * gate * sg
    if gate is not None:
        out['dgate'] = dy * core * sg * (1.0 + gate * (1.0 - sg))
    out['dweight'] = (dcore * n).reshape(-1, D).sum(0)
    out['dbias'] = dcore.reshape(-1, D).sum(0)
    dn = dcore * w
    dx = r * (dn - (dn.mean(-1, keepdim=True) if center else 0.0) - n * (dn * n).mean(-1, keepdim=True))
    out['dx'] = dx if dh is None else dx + dh
    out['terms'] = ((r * dn).norm() + (0.0 if dh is None else dh.norm())).item()  # size of what cancels in dx
    return out
