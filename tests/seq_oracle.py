"""64-bit statements of the token-sequence operators (linear attention with per-head decay, embedding) by their definitions, token by token,
and of the magnitudes that their rounding errors scale with."""
import torch


def _heads(x, H):
    return x.double().cpu().repeat_interleave(H // x.shape[-2], dim=-2)


def attend(q, k, v, g, state=None, lens=None, scale=None):
    """-> out [B,T,H,Dv], states [T+1 of B,H,Dk,Dv]"""
    B, T = q.shape[:2]
    H = g.shape[-1]
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    q, k, v = (_heads(x, H) for x in (q, k, v))
    a = torch.exp(g.double().cpu()).expand(B, T, H)
    n = torch.full((B,), T) if lens is None else lens.long().cpu().clamp(0, T)
    S = torch.zeros(B, H, q.shape[-1], v.shape[-1], dtype=torch.float64) if state is None else state.double().cpu()
    states, out = [S], torch.zeros(B, T, H, v.shape[-1], dtype=torch.float64)
    for t in range(T):
        on = (t < n).view(B, 1, 1, 1)
        new = a[:, t, :, None, None] * S + k[:, t, :, :, None] * v[:, t, :, None, :]
        S = torch.where(on, new, S)
        out[:, t] = torch.where(on[..., 0], (q[:, t, :, :, None] * S).sum(-2) * scale, torch.zeros(()).double())
        states.append(S)
    return out, states


def attend_grads(q, k, v, g, dout, state=None, lens=None, scale=None, dlast=None):
    """-> dq, dk, dv per shared head, dg [B,T,H], dstate; from the recurrences of the state and of its gradient"""
    B, T = q.shape[:2]
    H = g.shape[-1]
    hq, hk, hv = q.shape[2], k.shape[2], v.shape[2]
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    _, states = attend(q, k, v, g, state, lens, scale)
    q, k, v = (_heads(x, H) for x in (q, k, v))
    do = dout.double().cpu() * scale
    a = torch.exp(g.double().cpu()).expand(B, T, H)
    n = torch.full((B,), T) if lens is None else lens.long().cpu().clamp(0, T)
    E = torch.zeros_like(states[0]) if dlast is None else dlast.double().cpu()
    dq, dk, dv, dg = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v), torch.zeros(B, T, H, dtype=torch.float64)
    for t in reversed(range(T)):
        on = (t < n).view(B, 1, 1)
        dq[:, t] = torch.where(on, (states[t + 1] * do[:, t, :, None, :]).sum(-1), dq[:, t])
        F = E + q[:, t, :, :, None] * do[:, t, :, None, :]
        dk[:, t] = torch.where(on, (F * v[:, t, :, None, :]).sum(-1), dk[:, t])
        dv[:, t] = torch.where(on, (F * k[:, t, :, :, None]).sum(-2), dv[:, t])
        F = F * a[:, t, :, None, None]
        dg[:, t] = torch.where(on[..., 0], (F * states[t]).sum((-1, -2)), dg[:, t])
        E = torch.where(on[..., None], F, E)
    share = lambda x, h: x.reshape(B, T, h, H // h, -1).sum(3)
    return share(dq, hq), share(dk, hk), share(dv, hv), dg, E


def embed(ids, table, scale, pos=None):
    ids, table = ids.cpu().long(), table.double().cpu()
    ok = (ids >= 0) & (ids < table.shape[0])
    out = table[torch.where(ok, ids, torch.zeros(()).long())] * scale
    if pos is not None:
        out = out + pos.double().cpu()[: ids.shape[-1]]
    return torch.where(ok[..., None], out, torch.zeros(()).double())


def embed_grads(ids, dout, vocab, scale, pos_rows=None):
    T, D = dout.shape[-2:]
    ids, d = ids.cpu().long(), dout.double().cpu()
    ok = (ids >= 0) & (ids < vocab)
    d = torch.where(ok[..., None], d, torch.zeros(()).double())
    dtable = torch.zeros(vocab, D, dtype=torch.float64)
    dtable.index_add_(0, torch.where(ok, ids, torch.zeros(()).long()).reshape(-1), d.reshape(-1, D) * scale)
    dpos = None
    if pos_rows is not None:
        dpos = torch.zeros(pos_rows, D, dtype=torch.float64)
        dpos[:T] = d.reshape(-1, T, D).sum(0)
    return dtable, dpos
