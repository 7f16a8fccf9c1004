"""Linear attention with per-head decay (whole sequences, gradient, single tokens) and the token embedding on the GPU, against their 64-bit
definitions (seq_oracle).

Tolerances.  u = half a step of the output's type (fp32 2^-24, bf16 2^-8, fp16 2^-11 of the value).  An output is a sum of products; `mag` is
the same sum over the absolute values of its factors, so that a relative error e of every product moves the output by at most e * mag.
Products: each factor is exact or carries at most a few fp32 roundings and one exp (2^-21 together), the 16-bit kernels may hold an
intermediate factor (pair score, state) in two 8-bit pieces, off by at most 2^-17 of it, at most two such factors in a product.
Sums: at most n = Dk + Dv + 64 + T roundings of 2^-24 of a partial sum <= mag.
    |error| <= u |value| + (E + n 2^-24) mag,   E = 2^-21 for fp32, 2^-16 for 16-bit inputs (outputs kept in fp32 included)."""
import math
import threading

import pytest
import torch

import seq_oracle as O

pytestmark = pytest.mark.gpu
F32, BF, FP = torch.float32, torch.bfloat16, torch.float16
U = {F32: 2.0 ** -24, BF: 2.0 ** -8, FP: 2.0 ** -11}
E = {F32: 2.0 ** -21, BF: 2.0 ** -16, FP: 2.0 ** -16}


def ops():
    from v2a_hip import ops
    return ops


def near(got, want, mag, intype, n, what, times=1):
    got, want = got.detach().cpu(), want.cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    tol = times * (U[got.dtype] * want.abs() + (E[intype] + n * 2.0 ** -24) * mag.cpu()) + 1e-37
    if got.dtype == FP:
        tol = tol + 2.0 ** -25                 # fp16 subnormals: half a step
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    from conftest import parity_record
    parity_record(what, (err / tol).max().item() if err.numel() else 0.0, 1.0)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {(err / tol)[bad].max().item():.3g} tolerances, first at {bad.nonzero()[0].tolist()}"


def make(seed, B, T, H, Hq, Hk, Hv, Dk, Dv, dt, decay="token", state=True):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    q, k, v = r(B, T, Hq, Dk).to(dt), (r(B, T, Hk, Dk) * Dk ** -0.5).to(dt), r(B, T, Hv, Dv).to(dt)
    ld = -torch.nn.functional.softplus(r(H) - 3) if decay == "head" else -torch.nn.functional.softplus(2 * r(B, T, H) - 3)
    return dict(q=q, k=k, v=v, g=ld, state=r(B, H, Dk, Dv) if state else None, dout=r(B, T, H, Dv).to(dt), dlast=r(B, H, Dk, Dv))


def cu(x):
    return None if x is None else x.cuda()


def ab(x):
    return None if x is None else x.abs()


def check_fwd(c, lens=None, scale=None, got=None, what="fwd"):
    n = c["q"].shape[-1] + c["v"].shape[-1] + 64 + c["q"].shape[1]
    if got is None:
        got = ops().linear_attention_fwd(cu(c["q"]), cu(c["k"]), cu(c["v"]), cu(c["g"]), state=cu(c["state"]), lens=cu(lens), scale=scale, want_state=True)
    out, states = O.attend(c["q"], c["k"], c["v"], c["g"], c["state"], lens, scale)
    mag, mags = O.attend(ab(c["q"]), ab(c["k"]), ab(c["v"]), c["g"], ab(c["state"]), lens, None if scale is None else abs(scale))
    near(got[0], out, mag, c["q"].dtype, n, what + " out")
    near(got[1], states[-1], mags[-1], c["q"].dtype, n, what + " state")


def check_bwd(c, lens=None, scale=None, got=None, dlast=True, what="bwd"):
    B, T, H = c["dout"].shape[:3]
    dl = c["dlast"] if dlast else None
    dt = c["q"].dtype
    n = c["q"].shape[-1] + c["v"].shape[-1] + 64 + T
    if got is None:
        got = ops().linear_attention_bwd(cu(c["q"]), cu(c["k"]), cu(c["v"]), cu(c["g"]), cu(c["dout"]), state=cu(c["state"]), lens=cu(lens), scale=scale,
                                         dstate=cu(dl))
    dq, dk, dv, dg, ds = O.attend_grads(c["q"], c["k"], c["v"], c["g"], c["dout"], c["state"], lens, scale, dl)
    s1 = None if scale is None else abs(scale)
    m = O.attend_grads(ab(c["q"]), ab(c["k"]), ab(c["v"]), c["g"], ab(c["dout"]), ab(c["state"]), lens, s1, ab(dl))
    near(got[0], dq, m[0], dt, n, what + " dq")
    near(got[1], dk, m[1], dt, n, what + " dk")
    near(got[2], dv, m[2], dt, n, what + " dv")
    # d decay is a difference of running sums over the tokens of a chunk: their magnitude is that of sum |q_i . dq_i| + |k_j . dk_j| over the row
    per = lambda x, y: (torch.repeat_interleave(x.double().abs(), H // x.shape[2], 2) * y).sum(-1)
    full = O.attend_grads(*(torch.repeat_interleave(ab(c[x]).double(), H // c[x].shape[2], 2) for x in ("q", "k", "v")), c["g"], ab(c["dout"]), ab(c["state"]),
                          lens, s1, ab(dl))
    mg = (per(c["q"], full[0]) + per(c["k"], full[1])).sum(1, keepdim=True).expand(B, T, H) + m[3]
    if c["g"].dim() == 1:
        near(got[3], dg.sum((0, 1)), mg.sum((0, 1)), dt, n, what + " dg")
    else:
        near(got[3], dg, mg, dt, n, what + " dg")
    if c["state"] is None:
        assert got[4] is None
    else:
        near(got[4], ds, m[4], dt, n, what + " dstate")


# B, T, H, Hq, Hk, Hv, Dk, Dv, decay, state
SHAPES = [
    (1, 1, 1, 1, 1, 1, 1, 1, "head", False),
    (2, 1, 4, 4, 4, 4, 48, 48, "token", True),
    (3, 10, 4, 4, 4, 4, 16, 32, "head", False),
    (2, 15, 6, 2, 2, 6, 33, 17, "token", True),
    (1, 16, 2, 2, 2, 2, 64, 64, "token", True),
    (2, 63, 4, 4, 1, 1, 40, 72, "token", False),
    (1, 64, 3, 3, 3, 3, 128, 128, "head", True),
    (2, 65, 4, 1, 4, 2, 64, 100, "token", True),
    (1, 129, 2, 2, 1, 1, 128, 64, "token", True),
    (2, 200, 4, 2, 4, 4, 24, 128, "head", True),
    (1, 777, 2, 1, 1, 2, 40, 72, "token", True),
    (1, 1100, 1, 1, 1, 1, 128, 128, "token", False),
    (1, 320, 2, 2, 2, 2, 100, 33, "token", True),
    (1, 400, 3, 3, 1, 3, 33, 128, "head", True),
    (2, 260, 2, 1, 2, 2, 32, 20, "token", True),
    (1, 192, 2, 2, 2, 1, 80, 48, "token", True),
    (2, 900, 40, 40, 8, 40, 40, 36, "token", True),          # segments of four chunks
    (2, 333, 3, 3, 1, 3, 72, 96, "token", True), (1, 130, 2, 1, 2, 2, 96, 80, "head", True), (1, 450, 2, 2, 2, 1, 66, 91, "token", False),
]


@pytest.mark.parametrize("dt", [F32, BF, FP], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s[:8])))
def test_forward_and_gradient(shape, dt):
    B, T, H, Hq, Hk, Hv, Dk, Dv, decay, state = shape
    c = make(sum(shape[:8]), B, T, H, Hq, Hk, Hv, Dk, Dv, dt, decay, state)
    check_fwd(c)
    check_bwd(c, dlast=state or T % 2 == 0)


@pytest.mark.parametrize("dt", [F32, BF, FP], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("T", [9, 150, 640])
def test_padded_rows_are_not_read(T, dt):
    """Lengths 0, 1, T, past T and below 0; what is behind a row's end is NaN and infinity and must reach nothing."""
    lens = torch.tensor([T, 0, 1, T // 2 + 1, T + 5, -3], dtype=torch.int32)
    c = make(T, 6, T, 4, 4, 2, 4, 24, 40, dt)
    check_fwd(c, lens)
    clean = [ops().linear_attention_fwd(*(cu(c[x]) for x in ("q", "k", "v", "g")), state=cu(c["state"]), lens=lens.cuda(), want_state=True),
             ops().linear_attention_bwd(*(cu(c[x]) for x in ("q", "k", "v", "g", "dout")), state=cu(c["state"]), lens=lens.cuda(), dstate=cu(c["dlast"]))]
    check_bwd(c, lens, got=clean[1])
    for b, n in enumerate(lens.tolist()):
        n = min(max(n, 0), T)
        for x, bad in (("q", math.nan), ("k", math.inf), ("v", -math.inf), ("g", math.nan), ("dout", math.nan)):
            c[x][b, n:] = bad
    dirty = [ops().linear_attention_fwd(*(cu(c[x]) for x in ("q", "k", "v", "g")), state=cu(c["state"]), lens=lens.cuda(), want_state=True),
             ops().linear_attention_bwd(*(cu(c[x]) for x in ("q", "k", "v", "g", "dout")), state=cu(c["state"]), lens=lens.cuda(), dstate=cu(c["dlast"]))]
    for x, y in zip(clean[0] + clean[1], dirty[0] + dirty[1]):
        assert torch.equal(x, y)
    assert torch.equal(dirty[0][1][1].cpu(), c["state"][1]) and torch.equal(dirty[1][4][1].cpu(), c["dlast"][1])      # an empty row: the state passes through
    for b, n in enumerate(lens.tolist()):
        n = min(max(n, 0), T)
        for x in (dirty[0][0],) + dirty[1][:4]:
            assert not x[b, n:].any()


@pytest.mark.parametrize("dt", [F32, BF], ids=["fp32", "bf16"])
@pytest.mark.parametrize("low", [-math.inf, torch.finfo(F32).min, -200.0])
def test_decays_that_clear_the_state(low, dt):
    """exp of these is 0: what comes before the token reaches nothing after it, forwards or backwards, and the decay gets no gradient."""
    c = make(5, 2, 200, 2, 2, 2, 2, 32, 32, dt)
    at = [0, 1, 63, 64, 100, 101, 128, 199]
    c["g"][:, at] = low
    check_fwd(c)
    got = ops().linear_attention_bwd(*(cu(c[x]) for x in ("q", "k", "v", "g", "dout")), state=cu(c["state"]), dstate=cu(c["dlast"]))
    check_bwd(c, got=got)
    assert not got[4].any()
    a = [c[x][:, 100:].contiguous() for x in ("q", "k", "v", "g")]
    alone, _ = ops().linear_attention_fwd(*(cu(x) for x in a))
    both, _ = ops().linear_attention_fwd(*(cu(c[x]) for x in ("q", "k", "v", "g")), state=cu(c["state"]))
    # both are computed: |both - alone| <= |both - true| + |alone - true|, twice the bound (and the value the bound goes by is itself off by one
    # rounding u, which moves the bound by u^2 |value| <= 2^-16 |value| <= E mag of the 16-bit types, covered by the third)
    near(both[:, 100:], alone.double(), O.attend(*(ab(x) for x in a[:3]), a[3])[0], dt, 300, "after a reset", times=3)


@pytest.mark.parametrize("dt", [F32, BF, FP], ids=["fp32", "bf16", "fp16"])
def test_views_of_packed_projections(dt):
    """q, k, v as column blocks of one projection output, heads before tokens, a broadcast head, an odd first element: equal to contiguous."""
    B, T, H, D = 2, 70, 4, 24
    g = torch.Generator().manual_seed(1)
    big = torch.randn(B * T * 3 * H * D + 3, generator=g).to(dt).cuda()
    ld = (-torch.rand(H, T, B, generator=g)).cuda().permute(2, 1, 0)
    dout = torch.randn(B, H, T, D, generator=g).to(dt).cuda().transpose(1, 2)
    for off in (0, 1, 3):
        qkv = big[off:off + B * T * 3 * H * D].view(B, T, 3, H, D)
        views = [qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2]]
        odd = [views[0], views[1][:, :, :1].expand(B, T, H, D), views[2].transpose(1, 2).contiguous().transpose(1, 2)]
        for x in (views, odd):
            want = ops().linear_attention_fwd(*(y.contiguous() for y in x), ld.contiguous(), want_state=True)
            got = ops().linear_attention_fwd(*x, ld, want_state=True)
            assert all(torch.equal(a, b) for a, b in zip(want, got))
            want = ops().linear_attention_bwd(*(y.contiguous() for y in x), ld.contiguous(), dout.contiguous())
            got = ops().linear_attention_bwd(*x, ld, dout)
            assert all(torch.equal(a, b) for a, b in zip(want[:4], got[:4]))
        step = [y[:, 5] for y in views]
        S = torch.randn(B, H, D, D, generator=g).cuda()
        S1, S2 = S.clone(), S.clone()
        want = ops().linear_attention_step(*(y.contiguous() for y in step), ld[:, 5].contiguous(), S1)
        got = ops().linear_attention_step(*step, ld[:, 5], S2)
        assert torch.equal(want, got) and torch.equal(S1, S2)


def test_no_tokens_and_no_rows():
    S = torch.randn(2, 4, 8, 16).cuda()
    z = lambda B, T: (torch.zeros(B, T, 4, 8).cuda(), torch.zeros(B, T, 4, 8).cuda(), torch.zeros(B, T, 4, 16).cuda(), torch.zeros(4).cuda())
    out, last = ops().linear_attention_fwd(*z(2, 0), state=S, want_state=True)
    assert out.shape == (2, 0, 4, 16) and torch.equal(last, S)
    out, last = ops().linear_attention_fwd(*z(2, 0), want_state=True)
    assert not last.any()
    dq, dk, dv, dg, ds = ops().linear_attention_bwd(*z(2, 0), out, state=S, dstate=S)
    assert dq.shape == (2, 0, 4, 8) and not dg.any() and torch.equal(ds, S)
    out, last = ops().linear_attention_fwd(*z(0, 5), want_state=True)
    assert out.shape == (0, 5, 4, 16) and last.shape == (0, 4, 8, 16)
    dq, dk, dv, dg, ds = ops().linear_attention_bwd(*z(0, 5), out)
    assert dq.shape == (0, 5, 4, 8) and not dg.any() and ds is None
    assert ops().linear_attention_step(*(x[:, 0] if x.dim() == 4 else x for x in z(0, 5)), torch.zeros(0, 4, 8, 16).cuda()).shape == (0, 4, 16)


def test_long_sequences_of_no_rows():
    q, v, g = torch.zeros(0, 700, 4, 8).cuda(), torch.zeros(0, 700, 4, 16).cuda(), torch.zeros(4).cuda()
    assert ops().linear_attention_fwd(q, q, v, g)[0].shape == (0, 700, 4, 16)
    dq, dk, dv, dg, _ = ops().linear_attention_bwd(q, q, v, g, v)
    assert dq.shape == q.shape and dv.shape == v.shape and dg.shape == (4,) and not dg.any()


def check_step(c, t, S, slots=None, scale=None):
    """One call against the recurrence, rows of one slot in order."""
    B, H = c["q"].shape[0], c["g"].shape[-1]
    Dk, Dv = c["q"].shape[-1], c["v"].shape[-1]
    sc = Dk ** -0.5 if scale is None else scale
    want, mag = S.double().clone(), S.double().abs()
    wo, mo = torch.zeros(B, H, Dv, dtype=torch.float64), torch.zeros(B, H, Dv, dtype=torch.float64)
    q, k, v = (torch.repeat_interleave(c[x][:, t].double(), H // c[x].shape[2], 1) for x in ("q", "k", "v"))
    a = torch.exp(c["g"].double()).expand(B, c["q"].shape[1], H)[:, t]
    for b in range(B):
        s = b if slots is None else int(slots[b])
        if not 0 <= s < S.shape[0]:
            continue
        want[s] = a[b][:, None, None] * want[s] + k[b][:, :, None] * v[b][:, None, :]
        mag[s] = a[b][:, None, None] * mag[s] + (k[b][:, :, None] * v[b][:, None, :]).abs()
        wo[b] = (q[b][:, :, None] * want[s]).sum(1) * sc
        mo[b] = (q[b][:, :, None].abs() * mag[s]).sum(1) * abs(sc)
    Sg = S.cuda()
    g = c["g"] if c["g"].dim() == 1 else c["g"][:, t]
    out = ops().linear_attention_step(cu(c["q"][:, t]), cu(c["k"][:, t]), cu(c["v"][:, t]), cu(g), Sg, slots=cu(slots), scale=scale)
    near(out, wo, mo, c["q"].dtype if c["q"].dtype == F32 else F32, Dk + 8, "step out")      # products of 16-bit inputs and the fp32 state are fp32
    near(Sg, want, mag, F32, 8, "step state")
    return Sg


@pytest.mark.parametrize("dt", [F32, BF, FP], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1, 1, 1), (1, 8, 8, 8, 8, 48, 48), (5, 6, 2, 6, 3, 33, 17), (3, 4, 4, 1, 1, 128, 128), (2, 2, 2, 2, 2, 100, 64),
                                   (2, 2, 1, 2, 2, 16, 126), (2, 3, 3, 1, 3, 20, 33), (1, 2, 2, 2, 2, 65, 63), (3, 1, 1, 1, 1, 128, 65),
                                   (2, 2, 2, 2, 2, 3, 4)], ids=lambda s: "x".join(map(str, s)))
def test_step(shape, dt):
    B, H, Hq, Hk, Hv, Dk, Dv = shape
    c = make(sum(shape), B, 2, H, Hq, Hk, Hv, Dk, Dv, dt, "token" if B > 1 else "head")
    c["g"].flatten()[0] = -math.inf
    check_step(c, 0, c["state"])
    check_step(c, 1, c["state"], scale=-0.7)
    pool = torch.randn(2 * B + 1, H, Dk, Dv, generator=torch.Generator().manual_seed(2))
    slots = torch.randperm(2 * B + 1, generator=torch.Generator().manual_seed(3))[:B].int()
    check_step(c, 0, pool, slots)


def test_step_idle_rows_and_repeated_slots():
    """Slots -1, N, the smallest int: 0 and no state touched.  One slot named by many rows (300 rows: past one scan of a workgroup): successive tokens."""
    c = make(7, 300, 1, 2, 2, 1, 2, 12, 20, F32)
    pool = torch.randn(9, 2, 12, 20, generator=torch.Generator().manual_seed(2))
    slots = torch.randint(0, 9, (300,), generator=torch.Generator().manual_seed(4)).int()
    slots[::3] = 5
    slots[[4, 50, 299]] = torch.tensor([-1, 9, -2 ** 31], dtype=torch.int32)
    slots[slots == 7] = 6
    out = check_step(c, 0, pool, slots)
    assert torch.equal(out[7].cpu(), pool[7])
    bad = torch.full((300,), -1, dtype=torch.int32)
    c["k"][:] = math.nan
    S = pool.cuda()
    o = ops().linear_attention_step(cu(c["q"][:, 0]), cu(c["k"][:, 0]), cu(c["v"][:, 0]), cu(c["g"][:, 0]), S, slots=bad.cuda())
    assert not o.any() and torch.equal(S.cpu(), pool)


def test_step_on_a_pool_without_states():
    """N = 0: there is no slot to name, every row is idle."""
    c = make(7, 3, 1, 2, 2, 1, 2, 12, 20, F32)
    for slots in ([0, -1, 5], [2 ** 31 - 1, 0, 0]):
        o = ops().linear_attention_step(*(cu(c[x][:, 0]) for x in ("q", "k", "v", "g")), torch.zeros(0, 2, 12, 20).cuda(),
                                        slots=torch.tensor(slots, dtype=torch.int32).cuda())
        assert o.shape == (3, 2, 20) and not o.any()


@pytest.mark.parametrize("dt", [F32, BF, FP], ids=["fp32", "bf16", "fp16"])
def test_prompt_then_tokens_is_the_whole_sequence(dt):
    c = make(11, 3, 140, 6, 6, 2, 3, 48, 64, dt)
    a = [cu(c[x]) for x in ("q", "k", "v", "g")]
    cut = 133
    out, S = ops().linear_attention_fwd(*(x[:, :cut] for x in a), state=cu(c["state"]), want_state=True)
    outs = [out]
    for t in range(cut, 137):
        outs.append(ops().linear_attention_step(*(x[:, t] for x in a), S)[:, None])
    out, S = ops().linear_attention_fwd(*(x[:, 137:] for x in a), state=S, want_state=True)          # and a few tokens at once
    check_fwd(c, got=(torch.cat(outs + [out], 1), S), what="pieces")


def test_states_and_tokens_past_32_bit_offsets():
    """A state pool of more than 2^31 values, and q / k / v / dout whose rows lie more than 2^31 elements apart."""
    N = 2 ** 31 // (2 * 128 * 128) + 3
    pool = torch.empty(N, 2, 128, 128, device="cuda")
    c = make(3, 2, 1, 2, 2, 2, 2, 128, 128, BF)
    slots = torch.tensor([N - 1, 0], dtype=torch.int32)
    small = c["state"].clone()
    pool[N - 1], pool[0] = small[0].cuda(), small[1].cuda()
    ref = small.cuda()
    want = ops().linear_attention_step(*(cu(c[x][:, 0]) for x in ("q", "k", "v", "g")), ref)
    got = ops().linear_attention_step(*(cu(c[x][:, 0]) for x in ("q", "k", "v", "g")), pool, slots=slots.cuda())
    assert torch.equal(got, want) and torch.equal(pool[N - 1], ref[0]) and torch.equal(pool[0], ref[1])
    del pool
    big = torch.empty(2 ** 31 + 100000, dtype=BF, device="cuda")
    c = make(4, 2, 70, 2, 2, 2, 2, 32, 32, BF)
    far = {}
    for x in ("q", "k", "v", "dout"):
        far[x] = big.as_strided((2, 70, 2, 32), (2 ** 31 + 7, 64, 32, 1))
        far[x].copy_(c[x])
        a = [cu(c[y]) if y != x else far[x] for y in ("q", "k", "v", "g", "dout")]
        check_fwd(c, got=ops().linear_attention_fwd(*a[:4], state=cu(c["state"]), want_state=True), what="far " + x)
        check_bwd(c, got=ops().linear_attention_bwd(*a, state=cu(c["state"]), dstate=cu(c["dlast"])), what="far " + x)


def test_gradient_against_differences():
    """d loss along random directions, by differences of the 64-bit forward (step 1e-4: error ~1e-8), against the kernel's gradient of fp32
    inputs, off by at most (2^-21 + n 2^-24) of the sum of magnitudes as above."""
    c = make(21, 2, 90, 4, 2, 4, 2, 20, 28, F32)
    got = ops().linear_attention_bwd(*(cu(c[x]) for x in ("q", "k", "v", "g", "dout")), state=cu(c["state"]), dstate=cu(c["dlast"]))
    x = [c[y].double() for y in ("q", "k", "v", "g", "state")]

    def loss(y):
        out, S = O.attend(*y[:4], state=y[4])
        return ((out * c["dout"].double()).sum() + (S[-1] * c["dlast"].double()).sum()).item()

    g = torch.Generator().manual_seed(5)
    for i in range(5):
        d = torch.randn(x[i].shape, generator=g, dtype=torch.float64)
        up, down = list(x), list(x)
        up[i], down[i] = x[i] + 1e-4 * d, x[i] - 1e-4 * d
        diff = (loss(up) - loss(down)) / 2e-4
        dot = (got[i].double().cpu() * d).sum().item()
        assert abs(dot - diff) <= 1e-5 * (got[i].double().cpu() * d).abs().sum().item(), (i, dot, diff)


def _calls(c, S, slots):
    a = [c[x] for x in ("q", "k", "v", "g")]
    out, last = ops().linear_attention_fwd(*a, state=c["state"], want_state=True)
    grads = ops().linear_attention_bwd(*a, c["dout"], state=c["state"], dstate=c["dlast"])
    o = ops().linear_attention_step(*(x[:, 0] for x in a), S, slots=slots)
    return [out, last, *grads, o, S]


def _embed_calls(ids, table, pos, dout):
    out = ops().embed_fwd(ids, table, scale=1.5, pos=pos)
    return [out, *ops().embed_bwd(ids, dout, table.shape[0], scale=1.5, pos_rows=pos.shape[0])]


def _embed_inputs(seed, B=3, T=700, V=500, D=72, dt=BF):
    g = torch.Generator().manual_seed(seed)
    ids = (torch.rand(B, T, generator=g) ** 4 * V).long()
    return [ids.cuda(), torch.randn(V, D, generator=g).to(dt).cuda(), torch.randn(T + 2, D, generator=g).to(dt).cuda(), torch.randn(B, T, D, generator=g).to(dt).cuda()]


def test_captured_calls_replay():
    """All calls in one captured graph; replayed on changing inputs with eager calls and synchronizations between: every replay equals eager,
    bit for bit (all sums have a fixed order)."""
    sets = [make(s, 2, 600, 4, 2, 2, 4, 32, 64, BF) for s in (1, 2, 3)]
    sets = [{k: v.cuda() for k, v in c.items()} for c in sets]
    emb = [_embed_inputs(s) for s in (1, 2, 3)]
    slots = torch.tensor([3, 1], dtype=torch.int32, device="cuda")
    S0 = torch.randn(4, 4, 32, 64, generator=torch.Generator().manual_seed(1)).cuda()
    eager = [[y.clone() for y in _calls(c, S0.clone(), slots) + _embed_calls(*e)] for c, e in zip(sets, emb)]
    again = _calls(sets[0], S0.clone(), slots) + _embed_calls(*emb[0])
    assert all(torch.equal(x, y) for x, y in zip(eager[0], again))
    cur, cure, S = {k: v.clone() for k, v in sets[0].items()}, [x.clone() for x in emb[0]], S0.clone()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        res = _calls(cur, S, slots)
    with torch.cuda.graph(g2):
        rese = _embed_calls(*cure)
    for i in (0, 1, 2, 1, 0):
        for k in cur:
            cur[k].copy_(sets[i][k])
        for x, y in zip(cure, emb[i]):
            x.copy_(y)
        S.copy_(S0)
        g1.replay()
        g2.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(eager[i], res + rese)), i
        _calls(sets[(i + 1) % 3], S0.clone(), slots)


def test_two_streams_and_threads_at_once():
    sets = [{k: v.cuda() for k, v in make(s, 2, 500, 4, 4, 4, 4, 64, 64, FP).items()} for s in (1, 2)]
    emb = [_embed_inputs(s, B=8) for s in (1, 2)]
    slots = torch.tensor([1, 0], dtype=torch.int32, device="cuda")
    S0 = torch.randn(2, 4, 64, 64).cuda()
    want = [_calls(c, S0.clone(), slots) + _embed_calls(*e) for c, e in zip(sets, emb)]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        try:
            st = torch.cuda.Stream()
            with torch.cuda.stream(st):
                for _ in range(4):
                    got = _calls(sets[i], S0.clone(), slots) + _embed_calls(*emb[i])
                    st.synchronize()
                    if not all(torch.equal(x, y) for x, y in zip(want[i], got)):
                        bad.append(i)
                st.synchronize()
        except BaseException as e:      # noqa: a failure in a thread must fail the test
            bad.append(e)

    th = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    for t in th:
        t.start()
    for t in th:
        t.join()
    assert not bad, bad


# ---------------------------------------------------------------------------------------------- embedding
EMB = [  # ids shape, V, D, pos
    ((1,), 1, 1, True), ((1, 20), 1000, 512, True), ((3, 7), 5, 33, True), ((130,), 300, 50, False), ((2, 3, 41), 70, 96, True),
    ((9, 1031), 259, 40, False), ((4, 4100), 70000, 8, True), ((2, 600), 2, 257, False), ((5, 64), 65536, 16, False), ((40000,), 300, 12, True),
    ((8, 1000), 49408, 8, True), ((3000,), 7, 12, False), ((1500,), 9, 8, False), ((7, 300), 2 ** 20 + 3, 4, False), ((8192,), 1024, 8, False),
    ((8193,), 1023, 8, False), ((100,), 2 ** 21, 4, True),
]


@pytest.mark.parametrize("dt", [F32, BF, FP], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("shape,V,D,pos", EMB, ids=lambda s: str(s).replace(" ", "").replace("(", "").replace(")", ""))
def test_embedding_and_gradient(shape, V, D, pos, dt):
    """|error| <= u |value| + (2 + n) 2^-24 mag, n = tokens summed into a row (all in fp32)."""
    g = torch.Generator().manual_seed(V + D)
    ids = (torch.rand(shape, generator=g) ** 3 * V).long().clamp(max=V - 1)
    flat = ids.view(-1)
    if flat.numel() > 4:                    # empty places, and a token that fills a run longer than any tile
        flat[1], flat[-1], flat[2] = -1, V, 2 ** 40
        flat[flat.numel() // 2: flat.numel() // 2 + flat.numel() // 3] = V // 2
    T = shape[-1]
    table, dout = torch.randn(V, D, generator=g).to(dt), torch.randn(*shape, D, generator=g).to(dt)
    p = torch.randn(T + 3, D, generator=g).to(dt) if pos else None
    scale = D ** 0.5
    for i in (ids, ids.clamp(-1, V).int()):
        out = ops().embed_fwd(i.cuda(), table.cuda(), scale=scale, pos=cu(p))
        near(out, O.embed(ids, table, scale, p), O.embed(ids, table.abs(), scale, ab(p)), F32, 0, "embed")
        dtab, dpos = ops().embed_bwd(i.cuda(), dout.cuda(), V, scale=scale, pos_rows=T + 3 if pos else None)
        want, wp = O.embed_grads(ids, dout, V, scale, T + 3 if pos else None)
        mag, mp = O.embed_grads(ids, dout.abs(), V, scale, T + 3 if pos else None)
        near(dtab, want, mag, F32, flat.numel(), "dtable")
        if pos:
            near(dpos, wp, mp, F32, flat.numel() // T, "dpos")
        else:
            assert dpos is None
    assert not dtab[[r for r in range(min(V, 300)) if not (flat == r).any()]].any()


def test_embedding_of_views_and_of_nothing():
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(0, 50, (3, 17), generator=g).cuda()
    big = torch.randn(50 * 200 + 1, generator=g).cuda()
    for off, D in ((0, 64), (1, 64), (1, 33)):
        table = big[off:off + 50 * 200].view(50, 200)[:, 3:3 + D]
        pos = big[off:off + 20 * 200].view(20, 200)[:, 70:70 + D]
        assert torch.equal(ops().embed_fwd(ids, table, scale=0.5, pos=pos), ops().embed_fwd(ids, table.contiguous(), scale=0.5, pos=pos.contiguous()))
    assert ops().embed_fwd(ids[:0], table).shape == (0, 17, 33) and ops().embed_fwd(ids[:, :0].contiguous(), table).shape == (3, 0, 33)
    for empty in (ids[:0], ids[:, :0].contiguous()):
        dtab, dpos = ops().embed_bwd(empty, torch.zeros(*empty.shape, 33).cuda(), 50, pos_rows=17)
        assert not dtab.any() and not dpos.any() and dpos.shape == (17, 33)
    dout = torch.randn(3 * 17 * 64 + 1, generator=g).cuda()
    d1, d2 = dout[1:].view(3, 17, 64), dout[1:].clone().view(3, 17, 64)            # an odd first element: the same sums
    assert all(torch.equal(x, y) for x, y in zip(ops().embed_bwd(ids, d1, 50, pos_rows=17), ops().embed_bwd(ids, d2, 50, pos_rows=17)))
    none = torch.full((4, 5), -1).cuda()
    dtab, dpos = ops().embed_bwd(none, torch.full((4, 5, 33), math.nan).cuda(), 50, pos_rows=6)
    assert not dtab.any() and not dpos.any() and not ops().embed_fwd(none, table, pos=pos).any()


def test_token_hash_encoder_looks_up_the_same_values():
    from diffuser.libero.lb_train_utils import HashTextEncoder, HashTokenizer
    tok, enc = HashTokenizer(), HashTextEncoder(dim=64)
    ids = tok(["open the top drawer", "close it", ""])["input_ids"]
    want = enc(ids).last_hidden_state
    enc = enc.cuda()
    for x in (ids.cuda(), ids.t().contiguous().t().cuda(), ids):          # ids that stay on the host index the table on the GPU too
        assert torch.equal(enc(x).last_hidden_state.cpu(), want)


def test_embedding_past_32_bit_offsets():
    V = 2 ** 31 // 64 + 10
    table = torch.empty(V, 64, dtype=BF, device="cuda")
    table[V - 5:] = torch.arange(5, device="cuda")[:, None].to(BF)
    ids = torch.tensor([V - 1, V - 5, V - 2], device="cuda")
    assert torch.equal(ops().embed_fwd(ids, table)[:, 0].float().cpu(), torch.tensor([4.0, 0.0, 3.0]))
    del table
    dtab, _ = ops().embed_bwd(ids, torch.ones(3, 64, dtype=BF, device="cuda"), V)
    assert torch.equal(dtab[V - 5:, 63].float().cpu(), torch.tensor([1.0, 0, 0, 1, 1])) and not dtab[: V - 5].any()


# ---------------------------------------------------------------------------------------------- together
def test_a_recurrent_token_model_trains_and_serves():
    """Tokens -> embedding -> packed projection -> linear attention -> output, as a training step (loss gradient of every weight) and as a
    prompt followed by single tokens; fp32, against the same model in 64 bits through autograd (1e-5 of the largest gradient: the fp32 path
    of Linear is 1e-6)."""
    g = torch.Generator().manual_seed(9)
    V, D, H, B, T = 50, 64, 4, 2, 37
    hd = D // H
    ids = torch.randint(0, V, (B, T), generator=g)
    lens = torch.tensor([T, 20], dtype=torch.int32)
    W = {"table": torch.randn(V, D, generator=g) * 0.1, "pos": torch.randn(T, D, generator=g) * 0.1, "qkv": torch.randn(3 * D, D, generator=g) * D ** -0.5,
         "g": -torch.rand(H, generator=g)}
    R = torch.randn(B, T, H, hd, generator=g) * (torch.arange(T)[None, :, None, None] < lens[:, None, None, None])
    P = {k: v.double().requires_grad_() for k, v in W.items()}
    x = P["table"][ids] * D ** 0.5 + P["pos"]
    q, k, v = (x @ P["qkv"].T).view(B, T, 3, H, hd).unbind(2)
    i = torch.arange(T)
    w = torch.exp((i[:, None] - i[None]).clamp(min=0) * P["g"][:, None, None]) * (i[:, None] >= i[None])
    o = torch.einsum("hij,bhij,bjhd->bihd", w, torch.einsum("bihd,bjhd->bhij", q, k), v) * hd ** -0.5
    (o * R.double()).sum().backward()

    Wc = {k: v.cuda() for k, v in W.items()}
    x = ops().embed_fwd(ids.cuda(), Wc["table"], scale=D ** 0.5, pos=Wc["pos"])
    qkv = ops().linear(x.view(B * T, D), Wc["qkv"]).view(B, T, 3, H, hd)
    out, S = ops().linear_attention_fwd(*qkv.unbind(2), Wc["g"], lens=lens.cuda(), want_state=True)
    live = (torch.arange(T)[None] < lens[:, None])[..., None, None]
    rel = lambda a, b: ((a.double().cpu() - b).abs().max() / b.abs().max()).item()
    assert rel(out, o.detach() * live) <= 1e-5
    dq, dk, dv, dg, _ = ops().linear_attention_bwd(*qkv.unbind(2), Wc["g"], R.cuda(), lens=lens.cuda())
    dqkv = torch.stack([dq, dk, dv], 2).view(B * T, 3 * D)
    dW = dqkv.double().T @ x.view(B * T, D).double()
    dx = (dqkv @ Wc["qkv"]).view(B, T, D)
    dtable, dpos = ops().embed_bwd(ids.cuda(), dx, V, scale=D ** 0.5, pos_rows=T)
    for got, key in ((dtable, "table"), (dpos, "pos"), (dW, "qkv"), (dg, "g")):
        assert rel(got, P[key].grad) <= 1e-5, key
    # serving: the prompt's state, then each row's next tokens one by one
    for t in range(3):
        at = lens.long() + t
        tok = ids[torch.arange(B), at.clamp(max=T - 1)]
        y = ops().embed_fwd(tok.cuda().view(B, 1), Wc["table"], scale=D ** 0.5)[:, 0] + Wc["pos"][at.clamp(max=T - 1).cuda()]
        qkv1 = ops().linear(y, Wc["qkv"]).view(B, 3, H, hd)
        slots = torch.tensor([-1, 1], dtype=torch.int32, device="cuda")           # the first row has ended
        o1 = ops().linear_attention_step(*qkv1.unbind(1), Wc["g"], S, slots=slots)
        assert not o1[0].any() and rel(o1[1], o.detach()[1, 20 + t]) <= 1e-5
