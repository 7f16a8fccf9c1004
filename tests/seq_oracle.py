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


def decay_parts(q, k, v, g, dout, state=None, lens=None, scale=None, dlast=None, chunk=64):
    """Magnitude of what a chunk-wise sum for d decay adds up at each token -> [B,T,H]: for the chunk of `chunk` tokens that the token lies in,
    exp(G) <|S|, |E|> (state before the chunk, gradient of the one behind it), the products of its tokens with that state and that gradient,
    and twice its pair products (each is added in one row's sum and taken off in another's)."""
    B, T = q.shape[:2]
    H = g.shape[-1]
    scale = q.shape[-1] ** -0.5 if scale is None else abs(scale)
    q, k, v = (_heads(x, H).abs() for x in (q, k, v))
    do = dout.double().cpu().abs() * scale
    g = g.double().cpu().expand(B, T, H)
    n = torch.full((B,), T) if lens is None else lens.long().cpu().clamp(0, T)
    on = torch.arange(T)[None, :] < n[:, None]
    q, k, v, do = (torch.where(on[..., None, None], x, torch.zeros(()).double()) for x in (q, k, v, do))
    a = torch.where(on[..., None], torch.exp(g), torch.ones(()).double())
    S = torch.zeros(B, H, q.shape[-1], v.shape[-1], dtype=torch.float64) if state is None else state.double().cpu().abs()
    E = torch.zeros_like(S) if dlast is None else dlast.double().cpu().abs()
    before, behind, starts = [], {}, list(range(0, T, chunk))
    for t in range(T):
        if t % chunk == 0:
            before.append(S)
        S = a[:, t, :, None, None] * S + k[:, t, :, :, None] * v[:, t, :, None, :]
    for t in reversed(range(T)):
        if t == T - 1 or (t + 1) % chunk == 0:
            behind[t // chunk] = E
        E = a[:, t, :, None, None] * (E + q[:, t, :, :, None] * do[:, t, :, None, :])
    out = torch.zeros(B, T, H, dtype=torch.float64)
    for c, t0 in enumerate(starts):
        t1 = min(T, t0 + chunk)
        ac = a[:, t0:t1]
        L = t1 - t0
        W = torch.zeros(B, H, L, L, dtype=torch.float64)                       # decay from token j to token i, j <= i
        for i in range(L):
            W[:, :, i, i] = 1
            if i:
                W[:, :, i, :i] = W[:, :, i - 1, :i] * ac[:, i, :, None]
        head = torch.cumprod(ac, 1)                                            # from before the chunk to token i
        tail = W[:, :, -1].transpose(1, 2)                                     # from token j to the chunk's end
        qc, kc, vc, dc = (x[:, t0:t1] for x in (q, k, v, do))
        R = head * (torch.matmul(dc[:, :, :, None], before[c].transpose(-1, -2)[:, None])[..., 0, :] * qc).sum(-1)
        C = tail * (torch.matmul(vc[:, :, :, None], behind[c].transpose(-1, -2)[:, None])[..., 0, :] * kc).sum(-1)
        M = W * torch.einsum("bihd,bjhd->bhij", qc, kc) * torch.einsum("bihd,bjhd->bhij", dc, vc)
        Z = head[:, -1] * (before[c] * behind[c]).sum((-1, -2))
        out[:, t0:t1] = (Z + R.sum(1) + C.sum(1) + 2 * M.sum((-1, -2)))[:, None]
    return out
