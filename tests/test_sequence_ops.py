"""Refusals of the token-sequence operators (no GPU needed: every check precedes the launch) and the oracle's own gradient."""
import pytest
import torch

import seq_oracle as O


def _la(B=2, T=5, H=4, Hq=4, Hk=4, Hv=4, Dk=8, Dv=16, dt=torch.float32):
    return [torch.zeros(B, T, Hq, Dk, dtype=dt), torch.zeros(B, T, Hk, Dk, dtype=dt), torch.zeros(B, T, Hv, Dv, dtype=dt), torch.zeros(H)]


BAD = [
    ("need 4 dimensions", dict(), lambda a: a.__setitem__(0, a[0][0])),
    ("one type", dict(), lambda a: a.__setitem__(1, a[1].half())),
    ("one type", dict(dt=torch.float64), lambda a: None),
    ("different batch or length", dict(), lambda a: a.__setitem__(2, a[2][:, :3])),
    ("different head widths", dict(), lambda a: a.__setitem__(1, torch.zeros(2, 5, 4, 9))),
    ("1 to 128", dict(Dk=129), lambda a: None),
    ("1 to 128", dict(Dv=0), lambda a: None),
    ("q: last dimension", dict(), lambda a: a.__setitem__(0, a[0].transpose(2, 3).contiguous().transpose(2, 3))),
    ("v: last dimension", dict(), lambda a: a.__setitem__(2, torch.zeros(2, 5, 4, 32)[..., ::2])),
    ("log_decay: need fp32", dict(), lambda a: a.__setitem__(3, a[3].double())),
    ("log_decay: need fp32", dict(), lambda a: a.__setitem__(3, torch.zeros(2, 5, 4, 1))),
    ("log_decay: batch or length", dict(), lambda a: a.__setitem__(3, torch.zeros(2, 6, 4))),
    ("must divide", dict(Hk=3), lambda a: None),
    ("must divide", dict(Hv=8), lambda a: None),
    ("need CUDA", dict(), lambda a: None),
]


@pytest.mark.parametrize("msg,kw,change", BAD, ids=[f"{i}-{b[0].split()[0]}" for i, b in enumerate(BAD)])
def test_linear_attention_refuses(msg, kw, change):
    from v2a_hip import ops
    a = _la(**kw)
    change(a)
    with pytest.raises(ValueError, match=msg):
        ops.linear_attention_fwd(*a)
    with pytest.raises(ValueError, match=msg):
        ops.linear_attention_bwd(*a, torch.zeros(2, 5, 4, 16))
    if msg != "need 4 dimensions" and "length" not in msg:
        s = [x[:, 0] if x.dim() == 4 else x for x in a]
        with pytest.raises(ValueError, match=msg):
            ops.linear_attention_step(*s, torch.zeros(2, 4, 8, 16))


def test_operands_by_keyword():
    """The first operand may be named like the others: the call gets as far as the check for a GPU."""
    from v2a_hip import ops
    q, k, v, g = _la()
    ids = torch.zeros(2, 5, dtype=torch.int64)
    for call in (lambda: ops.linear_attention_fwd(q=q, k=k, v=v, log_decay=g), lambda: ops.linear_attention_fwd(k=k, v=v, log_decay=g, q=q),
                 lambda: ops.linear_attention_bwd(q=q, k=k, v=v, log_decay=g, dout=v),
                 lambda: ops.linear_attention_step(q=q[:, 0], k=k[:, 0], v=v[:, 0], log_decay=g, state=torch.zeros(2, 4, 8, 16)),
                 lambda: ops.embed_fwd(ids=ids, table=torch.zeros(7, 8)), lambda: ops.embed_bwd(ids=ids, dout=torch.zeros(2, 5, 8), vocab=7)):
        with pytest.raises(ValueError, match="need CUDA"):
            call()
    with pytest.raises(TypeError, match="'q'"):
        ops.linear_attention_fwd(k=k, v=v, log_decay=g)


def test_arguments_beside_the_operands_are_checked():
    """On the meta device: the same checks, past the one for a GPU."""
    from v2a_hip import ops

    class OnGpu(torch.Tensor):          # passes the device check; nothing is launched because a later check refuses
        is_cuda = True

    a = [x.as_subclass(OnGpu) for x in _la()]
    ok = torch.zeros(2, 4, 8, 16)
    for kw, msg in ((dict(state=ok[:1]), "state: need"), (dict(state=ok.double()), "state: need"), (dict(state=ok.transpose(2, 3)), "state: need"),
                    (dict(lens=torch.zeros(2)), "lens: need"), (dict(lens=torch.zeros(3, dtype=torch.int32)), "lens: need"),
                    (dict(lens=torch.zeros(2, dtype=torch.int64)), "lens: need")):
        with pytest.raises(ValueError, match=msg):
            ops.linear_attention_fwd.__wrapped__(*a, **kw)
    d = torch.zeros(2, 5, 4, 16)
    for dout, kw, msg in ((d[:, :4], {}, "dout: need"), (d.half(), {}, "dout: need"), (torch.zeros(2, 5, 4, 32)[..., ::2], {}, "dout: last"),
                          (d, dict(dstate=ok[:, :2]), "dstate: need"), (d, dict(state=ok[:, :2]), "state: need")):
        with pytest.raises(ValueError, match=msg):
            ops.linear_attention_bwd.__wrapped__(*a, dout, **kw)
    s = [x[:, 0] if x.dim() == 4 else x for x in a]
    for state, slots, msg in ((torch.zeros(3, 4, 8, 16), None, "one row per row"), (torch.zeros(3, 4, 8, 17), torch.zeros(2, dtype=torch.int32), "state: need"),
                              (torch.zeros(3, 4, 8, 16), torch.zeros(2, dtype=torch.int64), "lens: need"), (ok[0], None, "state: need")):
        with pytest.raises(ValueError, match=msg):
            ops.linear_attention_step.__wrapped__(*s, state, slots=slots)


def test_embedding_refuses():
    from v2a_hip import ops
    ids, table = torch.zeros(2, 3, dtype=torch.int64), torch.zeros(7, 8)
    for a, kw, msg in (((ids.float(), table), {}, "ids: need"), ((ids.t(), table), {}, "ids: need"), ((ids[0, 0], table), {}, "ids: need"),
                       ((ids, table), {}, "need CUDA")):
        with pytest.raises(ValueError, match=msg):
            ops.embed_fwd(*a, **kw)

    class OnGpu(torch.Tensor):
        is_cuda = True

    g = ids.as_subclass(OnGpu)
    for a, kw, msg in (((g, table.double()), {}, "table: need"), ((g, table[0]), {}, "table: need"), ((g, table.t()), {}, "table: last"),
                       ((g, table[:0]), {}, "table: need"), ((g, table), dict(pos=torch.zeros(2, 8)), "pos: need"),
                       ((g, table), dict(pos=torch.zeros(3, 8).half()), "pos: need"), ((g, table), dict(pos=torch.zeros(8, 3).t()), "pos: last")):
        with pytest.raises(ValueError, match=msg):
            ops.embed_fwd.__wrapped__(*a, **kw)
    d = torch.zeros(2, 3, 8)
    for a, kw, msg in (((g, d[:1], 7), {}, "dout: need"), ((g, d.double(), 7), {}, "dout: need"), ((g, d.transpose(0, 1).contiguous().transpose(0, 1), 7), {}, "dout: need"),
                       ((g, d, 0), {}, "vocab"), ((g, d, 2 ** 31), {}, "vocab"), ((g, d, 7), dict(pos_rows=2), "pos_rows")):
        with pytest.raises(ValueError, match=msg):
            ops.embed_bwd.__wrapped__(*a, **kw)


def test_c_entries_return_error_codes_before_any_launch():
    import ctypes
    from v2a_hip._lib import lib
    st = (ctypes.c_int64 * 15)()
    dims = (2, 8, 4, 4, 4, 4, 16, 16)
    null = [None] * 8
    assert lib.v2a_linattn_fwd(*null, st, *dims, 0, 1.0, None, 0, None) == -1
    assert lib.v2a_linattn_fwd(*null, None, *dims, 0, 1.0, None, 0, None) == -1
    assert lib.v2a_linattn_fwd(*null, st, 0, 8, 4, 4, 4, 4, 16, 16, 0, 1.0, None, 0, None) == 0        # no rows: nothing to do
    for bad in ((2, 8, 4, 3, 4, 4, 16, 16), (2, 8, 4, 4, 4, 4, 129, 16), (2, 8, 4, 4, 4, 4, 16, 0), (-1, 8, 4, 4, 4, 4, 16, 16), (2, -1, 4, 4, 4, 4, 16, 16),
                (1 << 20, 8, 4096, 4, 4, 4, 16, 16)):
        assert lib.v2a_linattn_fwd(*null, st, *bad, 0, 1.0, None, 0, None) == -1
        assert lib.v2a_linattn_bwd(*null, *[None] * 5, st, *bad, 0, 0, 1.0, None, 0, None) == -1
    assert lib.v2a_linattn_fwd(*null, st, *dims, 3, 1.0, None, 0, None) == -1
    assert lib.v2a_linattn_bwd(*null, *[None] * 5, st, *dims, 0, 0, 1.0, None, 0, None) == -1
    assert lib.v2a_linattn_step(*[None] * 7, st, 2, 2, 4, 4, 4, 4, 16, 16, 0, 1.0, None) == -1
    assert lib.v2a_linattn_step(*[None] * 7, st, 2, 1, 4, 4, 4, 4, 16, 16, 0, 1.0, None) == -1           # fewer states than rows, no slots
    assert lib.v2a_embed_fwd(None, 1, None, None, None, 6, 3, 7, 8, 8, 8, 0, 1.0, None) == -1
    assert lib.v2a_embed_fwd(None, 1, None, None, None, 5, 3, 7, 8, 8, 8, 0, 1.0, None) == -1            # not whole rows of T
    assert lib.v2a_embed_bwd(None, 1, None, None, None, 6, 3, 7, 8, 0, 0, 1.0, None, 0, None) == -1
    assert lib.v2a_embed_bwd(None, 1, None, None, None, 6, 3, 0, 8, 0, 0, 1.0, None, 0, None) == -1


def test_workspaces_of_long_calls_without_rows():
    from v2a_hip._lib import lib
    assert lib.v2a_linattn_fwd_workspace_bytes(0, 5000, 4, 64, 64, 1) == 0
    for T in (0, 1, 300, 5000):
        assert lib.v2a_linattn_bwd_workspace_bytes(0, T, 4, 4, 4, 4, 64, 64, 1, 1) == 0
    assert lib.v2a_linattn_bwd_workspace_bytes(1, 5000, 4, 4, 4, 4, 64, 64, 1, 1) > 0


def test_oracle_gradient_against_differences():
    """The oracle's hand-written gradient against central differences of its own forward (fp64, step 1e-5: error ~1e-10 of the value)."""
    gen = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)
    B, T, H, Dk, Dv = 2, 7, 4, 3, 5
    x = [r(B, T, 2, Dk), r(B, T, 4, Dk), r(B, T, 1, Dv), -r(B, T, H).abs(), r(B, H, Dk, Dv)]
    lens = torch.tensor([7, 4])
    dout, dlast = r(B, T, H, Dv), r(B, H, Dk, Dv)

    def loss(y):
        out, S = O.attend(*y[:4], state=y[4], lens=lens)
        return (out * dout).sum() + (S[-1] * dlast).sum()

    grads = O.attend_grads(*x[:4], dout, state=x[4], lens=lens, dlast=dlast)
    for i, gr in enumerate(grads):
        d = r(*x[i].shape)
        up, down = list(x), list(x)
        up[i], down[i] = x[i] + 1e-5 * d, x[i] - 1e-5 * d
        want = (loss(up) - loss(down)) / 2e-5
        got = (gr * d).sum()
        assert abs(got - want) <= 1e-7 * (gr * d).abs().sum(), i


def test_a_refusal_of_slots_names_them():
    from v2a_hip import ops

    class OnGpu(torch.Tensor):
        is_cuda = True

    s = [x[:, 0].as_subclass(OnGpu) if x.dim() == 4 else x.as_subclass(OnGpu) for x in _la()]
    for slots in (torch.zeros(2, dtype=torch.int64), torch.zeros(3, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)[::2]):
        with pytest.raises(ValueError, match="slots"):
            ops.linear_attention_step.__wrapped__(*s, torch.zeros(3, 4, 8, 16), slots=slots)
