"""Measured calls of the token-sequence operators of v2a_hip.ops: linear attention with a decay for each head (chunked form for whole
sequences, its gradient, recurrent form for single tokens) and the embedding lookup with its gradient.

`run` computes a pass either with elementary torch operations (own = False) or with the framework's kernels (own = True)."""
import math
import os
import sys

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
CHUNK = 64


# ---------------------------------------------------------------------------------------------- cases
def _la(kind, name, B, T, H, Dk, Dv, dtype, Hq=0, Hk=0, Hv=0, decay="head", ragged=False, state=False, resets=False, pool=0):
    c = dict(name=name, kind=kind, B=B, T=T, H=H, Hq=Hq or H, Hk=Hk or H, Hv=Hv or H, Dk=Dk, Dv=Dv, dtype=dtype, decay=decay, ragged=ragged,
             state=state, resets=resets, pool=pool)
    if not name:
        del c["name"]
    return c


def _emb(kind, name, B, T, V, D, dtype, pos, hot):
    c = dict(name=name, kind=kind, B=B, T=T, V=V, D=D, dtype=dtype, pos=pos, hot=hot)
    if not name:
        del c["name"]
    return c


def listed():
    return [
        # one control tick of one rollout through a layer of the 384-wide, 8-head policy trunk: latency only
        _la("step", "step_tick", 1, 1, 8, 48, 48, "fp32"),
        # one token for 512 live rollouts out of a pool of 640 recurrent states, in no order
        _la("step", "step_pool", 512, 1, 16, 128, 128, "bf16", decay="token", pool=640),
        # a batch of action sequences of horizon 10 through the same trunk, as at each denoising step
        _la("prompt", "prompt_horizon", 64, 10, 8, 48, 48, "fp32"),
        # padded observation histories of several packed episodes (the decay resets the state where one begins), keys / values shared by 3 heads
        _la("prompt", "prompt_history", 3, 1237, 12, 64, 64, "fp16", Hk=4, Hv=4, decay="token", ragged=True, state=True, resets=True),
        # fp32 (the framework's default arithmetic), value heads wider than key heads
        _la("prompt", "prompt_fp32", 8, 2048, 8, 64, 128, "fp32"),
        # one long sequence, continued from a state
        _la("prompt", "prompt_long", 1, 32768, 8, 128, 128, "bf16", state=True),
        # training on action sequences: forward and backward
        _la("train", "train_horizon", 64, 16, 4, 64, 64, "fp32"),
        # training on padded pieces with the state carried in and its gradient carried out, queries / keys shared by 3 heads, odd sizes
        _la("train", "train_pieces", 5, 777, 6, 40, 72, "fp16", Hq=2, Hk=2, decay="token", ragged=True, state=True),
        # training on long sequences
        _la("train", "train_long", 4, 4096, 8, 128, 128, "bf16", decay="token"),
        # one task string through the text tower's table, with position codes
        _emb("embed", "embed_text", 1, 20, 49408, 512, "fp32", True, "zipf"),
        # a batch of token sequences: lookup and gradient of the table and of the position codes; half the tokens are padding
        _emb("embed_train", "embed_train_text", 64, 128, 49408, 512, "bf16", True, "half"),
        # discretised actions: a small table, long sequences, every row hot
        _emb("embed_train", "embed_train_actions", 61, 1031, 259, 384, "fp32", False, "zipf"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _heads(rng, H):
    divs = [h for h in range(1, H + 1) if H % h == 0]
    return [H if rng.random() < 0.6 else rng.choice(divs) for _ in range(3)]


def draw(rng):
    kind = rng.choice(["step", "prompt", "prompt", "train", "train", "embed", "embed_train", "embed_train"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if kind in ("embed", "embed_train"):
        D = rng.choice([8, 50, 64, 96, 257, 384, 512, 768, 1000])
        V = _log_int(rng, 2, 65536)
        T = _log_int(rng, 1, 1500)
        B = _log_int(rng, 1, max(1, min(128, 62891 * 384 // (T * max(D, 384)))))
        return _emb(kind, "", B, T, V, D, dtype, rng.random() < 0.5, rng.choice(["zipf", "half", "even"]))
    H = rng.choice([1, 2, 3, 4, 6, 8, 12, 16])
    dims = [16, 24, 32, 33, 40, 48, 64, 72, 80, 96, 100, 128]
    Dk, Dv = rng.choice(dims), rng.choice(dims)
    Hq, Hk, Hv = _heads(rng, H)
    decay = rng.choice(["head", "token"])
    if kind == "step":
        B = _log_int(rng, 1, 512)
        return _la(kind, "", B, 1, H, Dk, Dv, dtype, Hq, Hk, Hv, decay, pool=B + rng.randint(0, B) if rng.random() < 0.5 else 0)
    T = _log_int(rng, 1, 32768 if kind == "prompt" else 4096)
    # tokens x heads of the largest listed case of the kind; fp32 has half of that
    most = (262144 if kind == "prompt" else 131072) // (2 if dtype == "fp32" else 1)
    T = min(T, most // H)
    B = _log_int(rng, 1, max(1, min(256, most // (H * T))))
    return _la(kind, "", B, T, H, Dk, Dv, dtype, Hq, Hk, Hv, decay, ragged=rng.random() < 0.4, state=rng.random() < 0.5,
               resets=decay == "token" and rng.random() < 0.3)


def _lens(case):
    """Lengths of a padded batch: the first row is full, the fourth empty, the others spread between."""
    T = case["T"]
    return [0 if b == 3 else max(1, round(T * ((1.0 + 0.6180339887 * b) % 1.0 or 1.0))) for b in range(case["B"])]


# ---------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape, mul=1.0, dtype=dt):
        return (torch.randn(shape, generator=g, device=dev) * mul).to(dtype)

    s = {"case": case}
    B, T = case["B"], case["T"]
    if case["kind"] in ("embed", "embed_train"):
        V, D = case["V"], case["D"]
        s["table"] = randn(V, D, mul=0.5)
        s["pos"] = randn(T, D, mul=0.1) if case["pos"] else None
        s["scale"] = math.sqrt(D)
        u = torch.rand((B, T), generator=g, device=dev, dtype=torch.float64)
        ids = (u * V).long() if case["hot"] == "even" else (torch.exp(u * math.log(V + 1.0)) - 1.0).long()      # zipf: frequency ~ 1 / rank
        ids = ids.clamp_(0, V - 1)
        if case["hot"] == "half":        # the second half of every row is the last token, which pads
            ids[:, (T + 1) // 2:] = V - 1
        s["ids"] = ids
        if case["kind"] == "embed_train":
            s["dout"] = randn(B, T, D)
        return s
    H, Dk, Dv = case["H"], case["Dk"], case["Dv"]
    step = case["kind"] == "step"
    lead = (B,) if step else (B, T)
    s["q"] = randn(*lead, case["Hq"], Dk)
    s["k"] = randn(*lead, case["Hk"], Dk, mul=Dk ** -0.5)
    s["v"] = randn(*lead, case["Hv"], Dv)
    if case["decay"] == "head":          # half-lives from about 16 tokens up, the same range for any number of heads
        s["g"] = torch.log1p(-(2.0 ** -(4.5 + 5.0 * torch.rand(H, generator=g, device=dev))))
    else:
        s["g"] = -torch.nn.functional.softplus(randn(*lead, H, mul=1.5, dtype=torch.float32) - 3.0)
        if case["resets"]:
            s["g"][torch.rand(lead, generator=g, device=dev) < 1.0 / 200] = -math.inf
    rows = case["pool"] or B
    s["state"] = randn(rows, H, Dk, Dv, mul=0.5, dtype=torch.float32) if step or case["state"] else None
    s["slots"] = torch.randperm(rows, generator=g, device=dev)[:B].int() if case["pool"] else None
    s["lens"] = torch.tensor(_lens(case), dtype=torch.int32, device=dev) if case["ragged"] else None
    if case["kind"] == "train":
        s["dout"] = randn(B, T, H, Dv)
        s["dstate"] = randn(B, H, Dk, Dv, mul=0.5, dtype=torch.float32) if case["state"] else None
    return s


# ---------------------------------------------------------------------------------------------- plain forms
def _heads32(x, H):
    return x.float().repeat_interleave(H // x.shape[-2], dim=-2)


def _attend(q, k, v, g, state, lens, scale):
    """q [B,T,H,Dk], k [B,T,H,Dk], v [B,T,H,Dv] in 32 bits, g [H] or [B,T,H] -> out [B,T,H,Dv], last state [B,H,Dk,Dv]: products inside chunks
    of tokens under the decay between each pair, and a product over the chunks' own states for what comes from before the chunk."""
    B, T, H, Dk = q.shape
    Dv = v.shape[-1]
    C = min(CHUNK, T)
    N = -(-T // C)
    g = torch.clamp(g.double(), min=-1e3).expand(B, T, H)
    if lens is not None:
        valid = (torch.arange(T, device=q.device)[None, :] < lens[:, None])[..., None]
        q, k, v = (torch.where(valid[..., None], x, torch.zeros_like(x)) for x in (q, k, v))
        g = torch.where(valid, g, torch.zeros_like(g))
    pad = N * C - T
    q, k, v = (torch.nn.functional.pad(x, (0, 0, 0, 0, 0, pad)).reshape(B, N, C, H, -1).permute(0, 3, 1, 2, 4) for x in (q, k, v))
    G = torch.nn.functional.pad(g, (0, 0, 0, pad)).reshape(B, N, C, H).permute(0, 3, 1, 2).cumsum(-1)                  # [B,H,N,C]
    upper = torch.ones(C, C, dtype=torch.bool, device=q.device).triu(1)
    W = torch.exp((G[..., :, None] - G[..., None, :]).masked_fill(upper, -math.inf)).float()
    out = ((q @ k.transpose(-1, -2)) * W) @ v
    local = (k * torch.exp(G[..., -1:] - G).float()[..., None]).transpose(-1, -2) @ v                                 # [B,H,N,Dk,Dv]
    A = torch.nn.functional.pad(G[..., -1].cumsum(-1), (1, 0))                                                         # log decay from the start to chunk n
    later = torch.ones(N + 1, N, dtype=torch.bool, device=q.device).tril(-1)
    M = torch.exp((A[..., :, None] - A[..., None, 1:]).masked_fill(~later, -math.inf)).float()                        # [B,H,N+1,N]
    S = (M @ local.reshape(B, H, N, Dk * Dv)).reshape(B, H, N + 1, Dk, Dv)
    if state is not None:
        S = S + torch.exp(A).float()[..., None, None] * state[:, :, None]
    out = out + (q * torch.exp(G).float()[..., None]) @ S[:, :, :N]
    out = (out * scale).permute(0, 2, 3, 1, 4).reshape(B, N * C, H, Dv)[:, :T]
    return out, S[:, :, N]


def _embed(table, ids, scale, pos):
    out = table[ids] * scale
    return out if pos is None else out + pos[: ids.shape[1]]


def _run_plain(s):
    c = s["case"]
    dt = DTYPES[c["dtype"]]
    kind = c["kind"]
    if kind == "embed":
        return _embed(s["table"].float(), s["ids"], s["scale"], None if s["pos"] is None else s["pos"].float()).to(dt)
    if kind == "embed_train":
        out = _embed(s["table"].float(), s["ids"], s["scale"], None if s["pos"] is None else s["pos"].float()).to(dt)
        ids, order = torch.sort(s["ids"].reshape(-1))
        d = s["dout"].reshape(-1, c["D"])[order].double()
        inner = torch.nn.functional.pad(d, (0, 0, 0, -len(d) % 256)).view(-1, 256, c["D"]).cumsum(1)     # running sums within blocks, then over blocks
        total = inner + torch.nn.functional.pad(inner[:-1, -1].cumsum(0), (0, 0, 1, 0))[:, None]
        total = torch.nn.functional.pad(total.view(-1, c["D"]), (0, 0, 1, 0))
        ends = torch.searchsorted(ids, torch.arange(c["V"] + 1, device=ids.device))
        dtable = total[ends[1:]] - total[ends[:-1]]
        dpos = None if s["pos"] is None else s["dout"].float().sum(0).to(dt)
        return {"out": out, "dtable": (dtable * s["scale"]).to(dt), "dpos": dpos}
    H, scale = c["H"], c["Dk"] ** -0.5
    if kind == "step":
        q, k, v = (_heads32(s[x], H) for x in ("q", "k", "v"))
        rows = s["state"] if s["slots"] is None else s["state"][s["slots"].long()]
        new = rows * torch.exp(s["g"])[..., None, None] + k[..., :, None] * v[..., None, :]
        out = (q[..., :, None] * new).sum(-2) * scale
        if s["slots"] is None:
            s["state"].copy_(new)
        else:
            s["state"].index_copy_(0, s["slots"].long(), new)
        return {"out": out.to(dt), "state": s["state"]}
    if kind == "prompt":
        out, last = _attend(*(_heads32(s[x], H) for x in ("q", "k", "v")), s["g"], s["state"], s["lens"], scale)
        return {"out": out.to(dt), "state": last}
    leaves = [s[x].float().requires_grad_() for x in ("q", "k", "v")] + [s["g"].detach().requires_grad_()]
    if s["state"] is not None:
        leaves.append(s["state"].detach().requires_grad_())
    state = leaves[4] if s["state"] is not None else None
    with torch.enable_grad():
        out, last = _attend(*(_heads32(x, H) for x in leaves[:3]), leaves[3], state, s["lens"], scale)
        tops, grads = ([out], [s["dout"].float()]) if state is None else ([out, last], [s["dout"].float(), s["dstate"]])
        got = torch.autograd.grad(tops, leaves, grads)
    res = {"out": out.detach().to(dt), "dq": got[0].to(dt), "dk": got[1].to(dt), "dv": got[2].to(dt), "ddecay": got[3]}
    if state is not None:
        res["dstate"] = got[4]
    return res


# ---------------------------------------------------------------------------------------------- the framework's calls
def _ops():
    at = os.path.join(os.getcwd(), "video-to-action-release_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    from v2a_hip import ops
    return ops


def _run_own(s):
    ops = _ops()
    c = s["case"]
    kind = c["kind"]
    if kind == "embed":
        return ops.embed_fwd(s["ids"], s["table"], scale=s["scale"], pos=s["pos"])
    if kind == "embed_train":
        out = ops.embed_fwd(s["ids"], s["table"], scale=s["scale"], pos=s["pos"])
        dtable, dpos = ops.embed_bwd(s["ids"], s["dout"], c["V"], scale=s["scale"], pos_rows=None if s["pos"] is None else c["T"])
        return {"out": out, "dtable": dtable, "dpos": dpos}
    if kind == "step":
        out = ops.linear_attention_step(s["q"], s["k"], s["v"], s["g"], s["state"], slots=s["slots"])
        return {"out": out, "state": s["state"]}
    if kind == "prompt":
        out, last = ops.linear_attention_fwd(s["q"], s["k"], s["v"], s["g"], state=s["state"], lens=s["lens"], want_state=True)
        return {"out": out, "state": last}
    out, _ = ops.linear_attention_fwd(s["q"], s["k"], s["v"], s["g"], state=s["state"], lens=s["lens"])
    dq, dk, dv, dg, dstate = ops.linear_attention_bwd(s["q"], s["k"], s["v"], s["g"], s["dout"], state=s["state"], lens=s["lens"],
                                                      dstate=s["dstate"])
    res = {"out": out, "dq": dq, "dk": dk, "dv": dv, "ddecay": dg}
    if s["state"] is not None:
        res["dstate"] = dstate
    return res


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    e = BYTES[case["dtype"]]
    B, T, kind = case["B"], case["T"], case["kind"]
    if kind in ("embed", "embed_train"):
        N, D = B * T, case["D"]
        rows = min(N, case["V"])
        fwd = N * 8 + rows * D * e + N * D * e + (T * D * e if case["pos"] else 0)
        if kind == "embed":
            return {"bytes": fwd, "flops": 2 * N * D}
        return {"bytes": fwd + N * 8 + N * D * e + case["V"] * D * e + (T * D * e if case["pos"] else 0), "flops": 4 * N * D}
    H, Dk, Dv = case["H"], case["Dk"], case["Dv"]
    lens = _lens(case) if case["ragged"] else [T] * B
    live = sum(lens)
    per = case["Hq"] * Dk + case["Hk"] * Dk + case["Hv"] * Dv          # values of q, k, v a token has
    st = B * H * Dk * Dv * 4
    decay = 4 * H * (live if case["decay"] == "token" else 1)
    flops = sum(n * H * min(4 * Dk * Dv, (n + 1) * (Dk + Dv)) for n in lens)
    if kind == "step":
        return {"bytes": live * per * e + decay + 2 * st + B * H * Dv * e, "flops": 5 * B * H * Dk * Dv}
    fwd = live * per * e + decay + B * T * H * Dv * e + (st if case["state"] else 0)
    if kind == "prompt":
        return {"bytes": fwd + st, "flops": flops + 2 * live * H * Dk * Dv}
    bwd = live * per * e + decay + live * H * Dv * e + (3 * st if case["state"] else 0) + B * T * per * e + (4 * B * T * H if case["decay"] == "token" else 4 * H)
    return {"bytes": fwd + bwd, "flops": 3.5 * flops}


# ---------------------------------------------------------------------------------------------- 64-bit values
def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    B, T = case["B"], case["T"]
    if kind in ("embed", "embed_train"):
        V, D = case["V"], case["D"]
        ids = s["ids"].reshape(-1)
        out = torch.index_select(s["table"].double(), 0, ids).mul_(s["scale"]).view(B, T, D)
        if s["pos"] is not None:
            out += s["pos"].double()[None]
        if kind == "embed":
            return out
        dtable = torch.zeros((V, D), dtype=torch.float64, device=ids.device).index_add_(0, ids, s["dout"].double().view(-1, D))
        dpos = None if s["pos"] is None else s["dout"].double().sum(0)
        return {"out": out, "dtable": dtable * s["scale"], "dpos": dpos}
    H, Dk, Dv = case["H"], case["Dk"], case["Dv"]
    scale = Dk ** -0.5
    at = lambda x: torch.arange(H, device=x.device) // (H // x.shape[-2])          # the shared head that each head reads
    q, k, v = (s[x].double() for x in ("q", "k", "v"))
    hq, hk, hv = at(q), at(k), at(v)
    if kind == "step":
        rows = torch.arange(B, device=q.device) if s["slots"] is None else s["slots"].long()
        new = s["state"].double()
        upd = torch.exp(s["g"].double()).expand(B, H)[..., None, None] * new[rows] + torch.einsum("bhk,bhv->bhkv", k[:, hk], v[:, hv])
        new[rows] = upd
        return {"out": torch.einsum("bhk,bhkv->bhv", q[:, hq], upd) * scale, "state": new}
    a = torch.exp(s["g"].double()).expand(B, T, H)
    lens = torch.full((B,), T, device=q.device) if s["lens"] is None else s["lens"].long()
    live = torch.arange(T, device=q.device)[None, :] < lens[:, None]               # [B,T]
    zero = torch.zeros((), dtype=torch.float64, device=q.device)
    a = torch.where(live[..., None], a, zero + 1.0)
    q, k, v = (torch.where(live[..., None, None], x, zero) for x in (q, k, v))
    # the definition, token by token: S <- a_t S + k_t v_t^T, o_t = S^T q_t * scale
    S = torch.zeros((B, H, Dk, Dv), dtype=torch.float64, device=q.device) if s["state"] is None else s["state"].double()
    before, out = [], torch.empty((B, T, H, Dv), dtype=torch.float64, device=q.device)
    for t in range(T):
        if kind == "train":
            before.append(S)
        S = S * a[:, t, :, None, None] + k[:, t, hk, :, None] * v[:, t, hv, None, :]
        out[:, t] = torch.matmul(q[:, t, hq, None, :], S)[:, :, 0] * scale
    if kind == "prompt":
        return {"out": out, "state": S}
    d = torch.where(live[..., None, None], s["dout"].double(), zero) * scale
    dS = torch.zeros_like(S) if s["dstate"] is None else s["dstate"].double()
    dq, dk = (torch.zeros((B, T, H, Dk), dtype=torch.float64, device=q.device) for _ in range(2))
    dv, dg = torch.zeros((B, T, H, Dv), dtype=torch.float64, device=q.device), torch.zeros((B, T, H), dtype=torch.float64, device=q.device)
    for t in reversed(range(T)):
        dq[:, t] = torch.matmul(S, d[:, t, :, :, None])[..., 0]
        dS = dS + q[:, t, hq, :, None] * d[:, t, :, None, :]
        dk[:, t] = torch.matmul(dS, v[:, t, hv, :, None])[..., 0]
        dv[:, t] = torch.matmul(k[:, t, hk, None, :], dS)[:, :, 0]
        S = before.pop()
        dS = dS * a[:, t, :, None, None]
        dg[:, t] = (S * dS).sum((-1, -2)) * live[:, t, None]
    share = lambda x, like: x.view(B, T, like.shape[-2], H // like.shape[-2], -1).sum(3)
    res = {"out": out, "dq": share(dq, q), "dk": share(dk, k), "dv": share(dv, v), "ddecay": dg if s["g"].dim() == 3 else dg.sum((0, 1))}
    if s["state"] is not None:
        res["dstate"] = dS
    return res
