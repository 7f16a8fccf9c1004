"""d decay of linear attention, token by token, against a bound that goes by the token's own 64-token chunk.

The gradient kernel promises (its comment) a sum of the parts that cross each decay: what comes from before the chunk, what goes behind it, and
the chunk's own pairs.  Its error at a token then goes by the magnitude A of those parts (seq_oracle.decay_parts), whatever the rest of
the row holds:
    |error| <= u |value| + (2^-20 + 2 n 2^-24) A,   n = Dk + Dv + 64 + T,   u = 2^-24 (the output is fp32).
Inputs are held exactly in every type, and so are the state and its gradient as factors (fp32 or three 8-bit pieces); each carries one exp and a few
roundings (2^-21) and at most n roundings of 2^-24 of a partial sum no larger than its magnitude, and a part holds two such factors at most.
A difference of sums over the row, sum_{i >= t} (q_i . dq_i - k_i . dk_i), is the same number; its error goes by the row, and the rows below
hold tokens whose parts are 2^24 times as large as those of the tokens between them."""
import math

import pytest
import torch

import seq_oracle as O

F32, BF, FP = torch.float32, torch.bfloat16, torch.float16


def make(seed, B, T, H, Hq, Hk, Hv, Dk, Dv, dt, state=True):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    return dict(q=r(B, T, Hq, Dk).to(dt), k=(r(B, T, Hk, Dk) * Dk ** -0.5).to(dt), v=r(B, T, Hv, Dv).to(dt),
                g=-torch.nn.functional.softplus(2 * r(B, T, H) - 3), state=r(B, H, Dk, Dv) if state else None, dout=r(B, T, H, Dv).to(dt),
                dlast=r(B, H, Dk, Dv) if state else None)


def loud_and_quiet(dt, T=640, Dk=32, Dv=48):
    """Loud tokens (all four factors times 2^6, exact in every type) at both ends of the row, quiet ones between, with nothing carried over."""
    c = make(3, 1, T, 2, 2, 2, 2, Dk, Dv, dt, state=False)
    loud = torch.zeros(T, dtype=torch.bool)
    loud[:192] = loud[448:] = True
    for x in ("q", "k", "v", "dout"):
        c[x][:, loud] *= 64
    c["g"][:, [192, 448]] = -math.inf
    return c, loud


def bound(c, want, lens=None, scale=None):
    n = c["q"].shape[-1] + c["v"].shape[-1] + 64 + c["q"].shape[1]
    A = O.decay_parts(c["q"], c["k"], c["v"], c["g"], c["dout"], c["state"], lens, scale, c["dlast"])
    return 2.0 ** -24 * want.abs() + (2.0 ** -20 + 2 * n * 2.0 ** -24) * A + 1e-37


def exact(c, lens=None, scale=None):
    return O.attend_grads(c["q"], c["k"], c["v"], c["g"], c["dout"], c["state"], lens, scale, c["dlast"])


def test_the_parts_bound_their_sum():
    """|d decay| <= A, and A is 0 where nothing is: the parts are those of the definition."""
    c = make(5, 2, 150, 4, 2, 4, 1, 6, 10, F32)
    lens = torch.tensor([150, 70])
    A = O.decay_parts(c["q"], c["k"], c["v"], c["g"], c["dout"], c["state"], lens, None, c["dlast"])
    dg = exact(c, lens)[3]
    assert (dg.abs() <= A).all() and (A[0] > 0).all()
    c["state"] = c["dlast"] = None
    A = O.decay_parts(c["q"], c["k"], c["v"], c["g"], c["dout"], None, lens, None, None)
    assert (exact(c, lens)[3].abs() <= A).all() and not A[1, 128:].any()


@pytest.mark.parametrize("dt", [F32, BF, FP], ids=["fp32", "bf16", "fp16"])
def test_a_difference_of_sums_over_the_row_exceeds_the_bound(dt):
    """The same number formed from row-long fp32 sums, of gradients that are exact to fp32: far outside at the quiet tokens.  In 64 bits the two agree."""
    c, loud = loud_and_quiet(dt)
    dq, dk, _, dg, _ = exact(c)
    tol = bound(c, dg)
    per = (c["q"].double() * dq).sum(-1) - (c["k"].double() * dk).sum(-1)
    back = lambda x: x.flip(1).cumsum(1).flip(1)
    live = torch.isfinite(c["g"])
    assert ((back(per) - dg).abs() <= tol)[live].all()
    row = torch.zeros_like(per.float())
    s = torch.zeros_like(row[:, 0])
    for t in reversed(range(per.shape[1])):
        s = s + per[:, t].float()
        row[:, t] = s
    off = (row.double() - dg).abs() > tol
    quiet = (~loud)[None, :, None] & live
    assert off[quiet].float().mean() > 0.5


SHAPES = [(1, 1, 1, 1, 1, 1, 4, 4, True), (2, 65, 4, 1, 4, 2, 64, 100, True), (2, 200, 2, 2, 1, 1, 24, 128, True), (1, 777, 2, 1, 1, 2, 40, 72, True),
          (1, 1100, 1, 1, 1, 1, 128, 128, False), (2, 333, 3, 3, 1, 3, 72, 96, True), (2, 260, 2, 1, 2, 2, 32, 20, True), (3, 130, 2, 2, 2, 2, 64, 64, True)]


def check(c, lens=None, scale=None):
    from v2a_hip import ops
    cu = lambda x: None if x is None else x.cuda()
    got = ops.linear_attention_bwd(*(cu(c[x]) for x in ("q", "k", "v", "g", "dout")), state=cu(c["state"]), lens=cu(lens), scale=scale,
                                   dstate=cu(c["dlast"]))[3].cpu().double()
    want = exact(c, lens, scale)[3]
    tol = bound(c, want, lens, scale)
    err = (got - want).abs()
    from conftest import parity_record
    parity_record("d decay", (err / tol).max().item(), 1.0)
    assert (err <= tol).all(), ((err / tol).max().item(), (err > tol).nonzero()[0].tolist())


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, BF, FP], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s[:8])))
def test_every_token_within_the_bound_of_its_chunk(shape, dt):
    c = make(sum(shape[:8]), *shape[:8], dt, shape[8])
    check(c)
    if shape[0] > 1:
        check(c, torch.tensor([shape[1], shape[1] // 3 + 1, 0][:shape[0]], dtype=torch.int32), scale=-0.3)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, BF, FP], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("width", [(32, 48), (64, 64), (80, 96), (128, 128)], ids=str)
def test_quiet_tokens_between_loud_ones(width, dt):
    check(loud_and_quiet(dt, Dk=width[0], Dv=width[1])[0])
