"""The training operators on the GPU against their plain forms in 64 bits.

Bounds: U is the unit roundoff of a result's type, E32 that of the fp32 arithmetic before it;
each test says which roundings it counts."""

import pytest
import torch

import train_ref as R
from train_ref import E32, TINY, U, close

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
RNG = (0x1234_5678_9ABC_DEF0, 77)


@pytest.fixture(scope="module")
def T():
    from defmuon_amd import train_ops
    return train_ops


@pytest.fixture(scope="module")
def Err():
    from defmuon_amd._native import NativeError
    return NativeError


def normal(*shape, dtype=F32, std=1.0, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dtype)


def ids_of(shape, vocab, seed=0, kind="zipf"):
    g = torch.Generator().manual_seed(seed)
    if kind == "same":
        return torch.full(shape, vocab // 2)
    if kind == "flat":
        return torch.randint(0, vocab, shape, generator=g)
    u = torch.rand(shape, generator=g, dtype=torch.float64)
    return ((vocab + 1.0) ** u - 1).long().clamp(0, vocab - 1)


# ---- dropout ----------------------------------------------------------------------------------
# x * scale, the addition, the scale itself: three fp32 roundings, then the result's
def drop_bound(x, r, want, dtype):
    return 4 * E32 * (x.abs() + r.abs()) + 1.01 * U[dtype] * want.abs() + TINY[dtype]


@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 1.0])
@pytest.mark.parametrize("shape", [(), (1,), (7,), (1, 8), (3, 8), (5, 771), (64, 768),
                                   (2, 3, 5, 33), (257, 2050)])
@pytest.mark.parametrize("dtype,res", [(F32, None), (BF16, None), (F16, None), (BF16, F32),
                                       (F16, F16), (F32, BF16)])
def test_dropout(T, shape, dtype, res, p):
    x = normal(*shape, dtype=dtype)
    r = None if res is None else normal(*shape, dtype=res, seed=1)
    got = T.dropout(x.to(DEV), p, RNG, None if r is None else r.to(DEV))
    y = R.drop(x.double(), p, RNG)
    rd = torch.zeros(()).double() if r is None else r.double()
    want = y + rd
    assert got.dtype == (dtype if r is None else res)
    close(got, want, drop_bound(y, rd, want, got.dtype))
    back = T.dropout_backward(x.to(DEV), p, RNG, F32)
    close(back, y, drop_bound(y, y * 0, y, F32))


@pytest.mark.parametrize("layout", ["columns", "odd columns", "every other row", "transposed",
                                    "broadcast rows", "expanded scalar", "shifted"])
def test_dropout_of_strided_tensors(T, layout):
    base = normal(24, 96, seed=3)
    b = base.to(DEV)

    def view(t):
        return {"columns": lambda: t[:, 32:64], "odd columns": lambda: t[:, 5:38],
                "every other row": lambda: t[::2], "transposed": lambda: t.T,
                "broadcast rows": lambda: t[3].expand(7, 96),
                "expanded scalar": lambda: t[0, 0].expand(5, 13),
                "shifted": lambda: t.view(-1)[1:1 + 2000].view(40, 50)}[layout]()
    x, xg = view(base), view(b)
    want = R.drop(x.double(), 0.3, RNG)
    close(T.dropout(xg, 0.3, RNG), want, drop_bound(want, want * 0, want, F32))
    r = normal(*x.shape, seed=4).double()
    got = T.dropout(r.float().to(DEV), 0.3, RNG, residual=xg)
    y = R.drop(r, 0.3, RNG)
    close(got, y + x.double(), drop_bound(y, x.double(), y + x.double(), F32))


def test_dropped_elements_leave_nothing_behind(T):
    k = R.keep(0, 4096, 0.5, RNG)
    x = torch.where(k, torch.full((4096,), 2.0), torch.tensor(float("nan")))
    x[::3] = torch.where(k[::3], torch.tensor(2.0), torch.tensor(float("inf")))
    got = T.dropout(x.to(DEV), 0.5, RNG).cpu()
    assert torch.equal(got, torch.where(k, torch.tensor(4.0), torch.tensor(0.0)))
    x = torch.where(k, torch.tensor(float("nan")), torch.tensor(1.0))
    assert torch.equal(torch.isnan(T.dropout(x.to(DEV), 0.5, RNG).cpu()), k)


def test_dropout_keys(T):
    x = torch.ones(4096, device=DEV)

    def mask(rng, p=0.5):
        return T.dropout(x, p, rng).cpu() != 0
    for rng in [(0, 0), (-1, -1), (2 ** 64 - 1, 2 ** 64 - 1), (5, 2 ** 32), (2 ** 32, 5)]:
        assert torch.equal(mask(rng), R.keep(0, 4096, 0.5, rng)), rng
        state = torch.tensor([r - 2 ** 64 if r >= 2 ** 63 else r for r in rng], device=DEV)
        assert torch.equal(mask(state), mask(rng))
    assert mask((1, 2), 2.0 ** -18).all()
    assert int(mask((1, 2), 1 - 2.0 ** -16).sum()) <= 4


def test_dropout_past_32_bit_offsets(T):
    n = (1 << 32) + 24
    x = torch.ones(n, dtype=BF16, device=DEV)
    y = T.dropout(x, 0.25, RNG)
    for first in (0, (1 << 31) - 16, (1 << 32) - 16):
        k = R.keep(first, 40, 0.25, RNG)
        want = torch.where(k, torch.tensor(4 / 3).to(BF16), torch.tensor(0.0).to(BF16))
        assert torch.equal(y[first:first + 40].cpu(), want), first
    assert bool((y[-8:].cpu() != 0).equal(R.keep(n - 8, 8, 0.25, RNG)))


def test_dropout_gradient(T):
    x, r = normal(9, 77).to(DEV).requires_grad_(), normal(9, 77, seed=1).to(DEV).requires_grad_()
    g = normal(9, 77, seed=2)
    y = T.dropout(x, 0.2, RNG, residual=r)
    dx, dr = torch.autograd.grad(y, (x, r), g.to(DEV))
    want = R.drop(g.double(), 0.2, RNG)
    close(dx, want, drop_bound(want, want * 0, want, F32))
    assert torch.equal(dr.cpu(), g)
    # against differences: y is linear in x, so <g, y(x + d) - y(x)> = <dx, d> but for the
    # roundings of y (two of them, 693 terms of size below 8)
    d = normal(9, 77, seed=5).to(DEV)
    with torch.no_grad():
        diff = (T.dropout(x + d, 0.2, RNG, residual=r) - y.detach()).double()
    lhs, rhs = float((diff * g.to(DEV)).sum()), float((dx.double() * d).sum())
    assert abs(lhs - rhs) <= 693 * 16 * 8 * E32
    xb = normal(9, 77, dtype=BF16).to(DEV).requires_grad_()
    (db,) = torch.autograd.grad(T.dropout(xb, 0.2, RNG, residual=r.detach()), xb, g.to(DEV))
    assert db.dtype == BF16
    close(db, want, drop_bound(want, want * 0, want, BF16))


def test_dropout_module(T):
    m = T.Dropout(0.5)
    x = torch.ones(100, 100, device=DEV, requires_grad=True)
    torch.manual_seed(0)
    a, b = m(x), m(x)
    assert not torch.equal(a, b)
    torch.manual_seed(0)
    assert torch.equal(m(x), a)
    assert torch.equal(m.eval()(x, residual=x), x + x)
    m.train()
    torch.manual_seed(0)
    y = torch.utils.checkpoint.checkpoint(m, x, use_reentrant=False)
    (g,) = torch.autograd.grad(y.sum(), x)
    assert torch.equal(g, a.detach())   # the repeated forward pass drew the same mask


def test_dropout_refusals(T, Err):
    x = torch.ones(4, 8, device=DEV)
    for call in (lambda: T.dropout(x, -0.1, RNG), lambda: T.dropout(x, 1.1, RNG),
                 lambda: T.dropout(x, float("nan"), RNG), lambda: T.dropout(x, 0.1, None),
                 lambda: T.dropout(x, 0.1, (1,)), lambda: T.dropout(x.double(), 0.1, RNG),
                 lambda: T.dropout(x, 0.1, RNG, x[:2]), lambda: T.dropout(x, 0.1, RNG, x.cpu()),
                 lambda: T.dropout(x, 0.1, RNG, x.double()),
                 lambda: T.dropout(x, 0.1, torch.zeros(2, dtype=torch.int64)),
                 lambda: T.dropout(x, 0.1, torch.zeros(3, dtype=torch.int64, device=DEV)),
                 lambda: T.dropout(x, 0.1, torch.zeros(2, device=DEV)),
                 lambda: T.dropout_backward(x, 0.1, RNG, torch.float64)):
        with pytest.raises(Err):
            call()
    for shape in ((0,), (0, 8), (4, 0)):
        assert T.dropout(torch.ones(shape, device=DEV), 0.1, RNG).shape == shape


# ---- embedding --------------------------------------------------------------------------------
def embed_bound(ids, w, pos, positions, scale, p, want, dtype):
    size = R.embedding(ids, w.abs(), None if pos is None else pos.abs(), positions, abs(scale),
                       p, RNG)
    return 4 * E32 * size + 1.01 * U[dtype] * want.abs() + TINY[dtype]


@pytest.mark.parametrize("shape,vocab,dim", [((1, 1), 3, 1), ((1, 1), 50257, 768),
                                             ((2, 5), 7, 8), ((3, 41), 100, 771),
                                             ((4, 33), 1000, 64), ((9,), 50, 130)])
@pytest.mark.parametrize("dtype,out", [(F32, F32), (F32, BF16), (BF16, BF16), (BF16, F32),
                                       (F16, F16)])
@pytest.mark.parametrize("with_pos,scale,p", [(False, 1.0, 0.0), (True, 1.0, 0.1),
                                              (True, -3.5, 0.0), (False, 27.7, 0.5)])
def test_embedding(T, shape, vocab, dim, dtype, out, with_pos, scale, p):
    ids = ids_of(shape, vocab)
    w = normal(vocab, dim, dtype=dtype)
    pos = normal(shape[-1] + 3, dim, dtype=dtype, seed=1) if with_pos else None
    want = R.embedding(ids, w, pos, None, scale, p, RNG)
    got = T.embedding(ids.to(DEV), w.to(DEV), None if pos is None else pos.to(DEV), scale=scale,
                      dropout_p=p, rng=RNG, out_dtype=out)
    assert got.dtype == out
    close(got, want, embed_bound(ids, w, pos, None, scale, p, want, out))


def test_embedding_layouts(T):
    w, pos = normal(50, 96), normal(20, 96, seed=1)
    ids = ids_of((6, 20), 50, kind="flat")
    positions = ids_of((6, 20), 20, seed=2, kind="flat")
    for i, p in ((ids, positions), (ids.int(), positions.int()), (ids.int(), positions),
                 (ids[:, ::2], positions[:, ::2]), (ids[:, :-1], positions[:, 1:]),
                 (ids.T, positions.T)):
        for wv, pv in (((slice(None), slice(0, 96)),) * 2, ((slice(None), slice(3, 40)),) * 2,
                       ((slice(None, None, 2), slice(8, 72)), (slice(None), slice(16, 80)))):
            ww, pp = w[wv], pos[pv]
            i2, ps = i % ww.shape[0], p
            got = T.embedding(i2.to(DEV), w.to(DEV)[wv], pos.to(DEV)[pv], positions=ps.to(DEV))
            want = R.embedding(i2, ww, pp, ps)
            close(got, want, embed_bound(i2, ww, pp, ps, 1.0, 0.0, want, F32))
    got = T.embedding(ids.to(DEV), w.to(DEV).T.contiguous().T)
    assert torch.equal(got.cpu(), w[ids])


def test_ids_outside_the_table(T):
    w = normal(10, 24).to(DEV)
    ids = torch.tensor([3, -1, 10, 9, 2 ** 40, -2 ** 40, 0])
    bad = torch.tensor([False, True, True, False, True, True, False])
    y = T.embedding(ids.to(DEV), w, dropout_p=0.5, rng=RNG).cpu()
    assert torch.equal(torch.isnan(y).all(1), bad) and not torch.isnan(y[~bad]).any()
    pos = normal(4, 24).to(DEV)
    t = torch.tensor([0, 1, 2, -1, 0, 0, 4])
    y = T.embedding(ids.to(DEV), w, pos, positions=t.to(DEV)).cpu()
    assert torch.isnan(y).all(1).tolist() == [False, True, True, True, True, True, True]
    g = normal(7, 24)
    dw, dp = T.embedding_backward(g.to(DEV), ids.to(DEV), 10, pos_rows=4, positions=t.to(DEV))
    for got, idx, rows in ((dw, ids, 10), (dp, t, 4)):
        want, size, n = R.table_grad(g, idx, rows)
        close(got, want, grad_bound(want, size, n, F32))


# n terms summed in fp32 in any order, the scales of dropout and the table, then the result's
def grad_bound(want, size, n, dtype):
    return (n + 8) * E32 * size + 1.01 * U[dtype] * want.abs() + TINY[dtype]


@pytest.mark.parametrize("tokens,vocab,dim,kind", [
    (1, 5, 1, "flat"), (2, 1, 8, "flat"), (63, 7, 24, "flat"), (64, 1000, 33, "flat"),
    (256, 40, 136, "same"), (255, 90, 1036, "zipf"),
    (257, 300, 771, "zipf"), (1000, 100, 64, "same"), (2049, 50257, 192, "zipf"),
    (5000, 70000, 40, "zipf"), (8192, 50257, 64, "zipf"), (8193, 1009, 96, "zipf"),
    (20001, 131072, 72, "zipf"), (40000, 17, 136, "flat"), (66000, 70001, 16, "same"),
    (300000, 50257, 8, "zipf")])
@pytest.mark.parametrize("dtype,out,p", [(F32, F32, 0.0), (BF16, F32, 0.1), (F16, F16, 0.0),
                                         (F32, BF16, 0.25)])
def test_embedding_gradient(T, tokens, vocab, dim, kind, dtype, out, p):
    ids = ids_of((tokens,), vocab, kind=kind)
    if tokens > 100 and kind != "same":
        ids[-tokens // 8:] = min(2, vocab - 1)   # padding
    pad = None if tokens < 100 else min(2, vocab - 1)
    g = normal(tokens, dim, dtype=dtype)
    args = dict(scale=1.5, padding_idx=pad, dropout_p=p, rng=RNG, dtype=out)
    dw, dp = T.embedding_backward(g.to(DEV), ids.to(DEV), vocab, **args)
    again, _ = T.embedding_backward(g.to(DEV), ids.to(DEV), vocab, **args)
    assert dp is None and dw.dtype == out
    assert torch.equal(dw, again)
    want, size, n = R.table_grad(g, ids, vocab, 1.5, p, RNG, pad)
    close(dw, want, grad_bound(want, size, n, out))


def test_gradient_of_a_table_of_many_rows(T):
    """Ids of 25 bits: four passes of the sort."""
    rows, tokens, dim = (1 << 24) + 9, 9001, 8
    ids = ids_of((tokens,), rows, kind="flat")
    ids[::7], ids[5], ids[11] = ids[0], rows - 1, rows
    g = normal(tokens, dim)
    dw, _ = T.embedding_backward(g.to(DEV), ids.to(DEV), rows)
    named, place = torch.unique(ids, return_inverse=True)
    want, size, n = R.table_grad(g, place, len(named))
    inside = named < rows
    named, want, bound = named[inside], want[inside], grad_bound(want, size, n, F32)[inside]
    close(dw[named.to(DEV)], want, bound)
    assert int(dw.ne(0).any(1).sum()) == len(named)


@pytest.mark.parametrize("batch,seq,rows,dim", [(1, 1, 1, 8), (1, 9, 16, 24), (8, 128, 128, 96),
                                                (300, 3, 5, 40), (2000, 1, 1, 520),
                                                (33, 70, 200, 17)])
@pytest.mark.parametrize("dtype,out,p", [(F32, F32, 0.0), (BF16, F32, 0.1), (F16, F16, 0.0)])
def test_position_gradient(T, batch, seq, rows, dim, dtype, out, p):
    ids = ids_of((batch, seq), 11)
    g = normal(batch, seq, dim, dtype=dtype)
    dw, dp = T.embedding_backward(g.to(DEV), ids.to(DEV), 0, pos_rows=rows, dropout_p=p, rng=RNG,
                                  scale=3.0, dtype=out)
    assert dw is None
    t = torch.arange(seq).expand(batch, seq)
    want, size, n = R.table_grad(g, t, rows, 1.0, p, RNG)
    close(dp, want, grad_bound(want, size, n, out))
    # the same positions, given
    _, dq = T.embedding_backward(g.to(DEV), ids.to(DEV), 0, pos_rows=rows, dropout_p=p, rng=RNG,
                                 positions=t.to(DEV), dtype=out)
    close(dq, want, grad_bound(want, size, n, out))


@pytest.mark.parametrize("batch", [1, 9])
@pytest.mark.parametrize("dim", [1, 5, 13, 72, 515, 519, 1031])
@pytest.mark.parametrize("out,p", [(F32, 0.0), (BF16, 0.0), (F32, 0.2)])
def test_gradients_are_added(T, batch, dim, out, p):
    seq = 250
    ids = ids_of((batch, seq), 300)
    g = normal(batch, seq, dim)
    w0, p0 = normal(300, dim, dtype=out, seed=5), normal(512, dim, dtype=out, seed=6)
    w, pg = w0.to(DEV), p0.to(DEV)
    dw, dp = T.embedding_backward(g.to(DEV), ids.to(DEV), 300, pos_rows=512, scale=2.0,
                                  weight_grad=w, pos_grad=pg, dropout_p=p, rng=RNG)
    assert dw is w and dp is pg
    want, size, n = R.table_grad(g, ids, 300, 2.0, p, RNG)
    close(w, want + w0.double(), grad_bound(want + w0.double(), size + w0.abs(), n, out))
    untouched = n[:, 0] == 0
    assert untouched.any() and torch.equal(w.cpu()[untouched], w0[untouched])
    want, size, n = R.table_grad(g, torch.arange(seq).expand(batch, seq), 512, 1.0, p, RNG)
    close(pg, want + p0.double(), grad_bound(want + p0.double(), size + p0.abs(), n, out))
    assert torch.equal(pg.cpu()[seq:], p0[seq:])


def test_gradient_of_strided_output(T):
    ids = ids_of((5, 30), 40)
    base = normal(5, 30, 100, seed=1)
    for view in (lambda t: t[..., 10:74], lambda t: t[..., 3:20], lambda t: t[:1].expand(5, 30, 100),
                 lambda t: t[0, 0].expand(5, 30, 100), lambda t: t[0, 0, 0].expand(5, 30, 9)):
        g = view(base)
        dw, dp = T.embedding_backward(view(base.to(DEV)), ids.to(DEV), 40, pos_rows=30,
                                      dropout_p=0.2, rng=RNG)
        want, size, n = R.table_grad(g, ids, 40, 1.0, 0.2, RNG)
        close(dw, want, grad_bound(want, size, n, F32))
        want, size, n = R.table_grad(g, torch.arange(30).expand(5, 30), 30, 1.0, 0.2, RNG)
        close(dp, want, grad_bound(want, size, n, F32))


def test_non_finite_gradients_stay_in_their_rows(T):
    ids = torch.tensor([4, 1, 4, 2, 0, 4])
    g = normal(6, 16)
    g[0, 3], g[3, 5], g[4] = float("nan"), float("inf"), float("nan")
    dw, _ = T.embedding_backward(g.to(DEV), ids.to(DEV), 6, padding_idx=0)
    want, size, n = R.table_grad(g, ids, 6, padding=0)
    close(dw, want, torch.nan_to_num(grad_bound(want, size, n, F32), 0.0, 0.0))


def test_embedding_of_no_tokens(T):
    w = normal(5, 8).to(DEV)
    none = torch.zeros((2, 0), dtype=torch.int64, device=DEV)
    assert T.embedding(none, w, w).shape == (2, 0, 8)
    dw, dp = T.embedding_backward(torch.zeros((2, 0, 8), device=DEV), none, 5, pos_rows=3)
    assert dw.shape == (5, 8) and dp.shape == (3, 8)
    assert not dw.any() and not dp.any()


def test_tables_past_32_bit_offsets(T):
    rows, dim = (1 << 20) + 5, 2048 + 8   # 2^31 elements and more
    w = torch.empty((rows, dim), dtype=BF16, device=DEV)
    w[-2:] = 3.0
    w[0] = 1.0
    ids = torch.tensor([rows - 1, 0, rows - 2], device=DEV)
    assert T.embedding(ids, w)[:, ::500].float().mean(1).tolist() == [3.0, 1.0, 3.0]
    del w
    g = normal(3, dim, dtype=BF16)
    dw, _ = T.embedding_backward(g.to(DEV), ids, rows, dtype=BF16)
    assert torch.equal(dw[[-1, 0, -2]].cpu(), g)
    assert not dw[1:5].any() and not dw[-5:-2].any() and not dw[rows // 2].any()


def test_embedding_autograd(T):
    w = normal(60, 40).to(DEV).requires_grad_()
    pos = normal(25, 40, seed=1).to(DEV).requires_grad_()
    ids, g = ids_of((3, 25), 60), normal(3, 25, 40, seed=2)
    y = T.embedding(ids.to(DEV), w, pos, scale=2.5, padding_idx=1, dropout_p=0.3, rng=RNG)
    dw, dp = torch.autograd.grad(y, (w, pos), g.to(DEV), retain_graph=True)
    want, size, n = R.table_grad(g, ids, 60, 2.5, 0.3, RNG, padding=1)
    close(dw, want, grad_bound(want, size, n, F32))
    want, size, n = R.table_grad(g, torch.arange(25).expand(3, 25), 25, 1.0, 0.3, RNG)
    close(dp, want, grad_bound(want, size, n, F32))
    (only,) = torch.autograd.grad(y, pos, g.to(DEV))
    assert torch.equal(only, dp)
    # against differences: linear in both tables (3000 terms below 64, two roundings)
    dW, dP = normal(60, 40, seed=7).to(DEV), normal(25, 40, seed=8).to(DEV)
    dW[1] = 0   # the padding row's gradient is zero by definition
    with torch.no_grad():
        y2 = T.embedding(ids.to(DEV), w + dW, pos + dP, scale=2.5, dropout_p=0.3, rng=RNG)
    lhs = float(((y2 - y.detach()).double() * g.to(DEV)).sum())
    rhs = float((dw.double() * dW).sum() + (dp.double() * dP).sum())
    assert abs(lhs - rhs) <= 3000 * 64 * 8 * E32
    # a table in half precision keeps its type
    h = w.detach().to(BF16).requires_grad_()
    (dh,) = torch.autograd.grad(T.embedding(ids.to(DEV), h, out_dtype=F32), h, g.to(DEV))
    want, size, n = R.table_grad(g, ids, 60)
    assert dh.dtype == BF16
    close(dh, want, grad_bound(want, size, n, BF16))


def test_embedding_refusals(T, Err):
    w = torch.ones(10, 8, device=DEV)
    ids = torch.zeros((2, 4), dtype=torch.int64, device=DEV)
    g = torch.ones(2, 4, 8, device=DEV)
    for call in (lambda: T.embedding(ids, w[0]), lambda: T.embedding(ids.float(), w),
                 lambda: T.embedding(ids.cpu(), w), lambda: T.embedding(ids, w.double()),
                 lambda: T.embedding(ids, w, w[:3]), lambda: T.embedding(ids, w, w[:, :4]),
                 lambda: T.embedding(ids, w, w.half()), lambda: T.embedding(ids, w, w.cpu()),
                 lambda: T.embedding(ids, w, positions=ids),
                 lambda: T.embedding(ids, w, w, positions=ids[0]),
                 lambda: T.embedding(ids, w, w, positions=ids.float()),
                 lambda: T.embedding(ids, w, padding_idx=10),
                 lambda: T.embedding(ids, w, padding_idx=-1),
                 lambda: T.embedding(ids, w, out_dtype=torch.float64),
                 lambda: T.embedding(ids, w, dropout_p=0.5),
                 lambda: T.embedding(ids, w, dropout_p=2.0, rng=RNG),
                 lambda: T.embedding(ids[0, 0], w, w),
                 lambda: T.embedding_backward(g[0], ids, 10),
                 lambda: T.embedding_backward(g, ids, -1),
                 lambda: T.embedding_backward(g, ids.float(), 10),
                 lambda: T.embedding_backward(g, ids, 10, pos_rows=3),
                 lambda: T.embedding_backward(g, ids, 10, padding_idx=10),
                 lambda: T.embedding_backward(g, ids, 10, dtype=torch.int32),
                 lambda: T.embedding_backward(g, ids, 10, weight_grad=w[:9]),
                 lambda: T.embedding_backward(g, ids, 10, weight_grad=w.double()),
                 lambda: T.embedding_backward(g, ids, 8, weight_grad=w[:8].T),
                 lambda: T.embedding_backward(g.double(), ids, 10)):
        with pytest.raises(Err):
            call()


# ---- cross entropy ----------------------------------------------------------------------------
class Xent:
    """The plain losses and gradient of a case, and their bounds.

    Counted: exponents of size d = max z - z carry three roundings (3 d E32), each exponential
    two; no lane adds more than max(64, V / 256) of them in sequence, and 32 more roundings
    join lanes and take the logarithm.  A loss adds four roundings of its terms' sizes."""

    def __init__(self, z, y, eps=0.0, zeta=0.0, ignore=-100):
        self.loss, self.dz, lse = R.xent(z, y, ignore, eps, zeta)
        zd, v = z.double(), z.shape[-1]
        fin = torch.isfinite(zd)
        size = torch.where(fin, zd.abs(), 0.0).amax(-1)
        m = torch.where(fin, zd, -1e30).amax(-1, keepdim=True)
        depth = torch.where(fin, m - zd, 0.0)
        rho = (max(64, v // 256) + 32 + 4 * depth.amax(-1)) * E32
        lse = torch.nan_to_num(lse, 0.0, 0.0, 0.0)
        self.lse_err = rho + 4 * E32 * (size + lse.abs())
        self.loss_err = (self.lse_err * (1 + 2 * zeta * lse.abs())
                         + 4 * E32 * (2 * size + lse.abs() + zeta * lse ** 2)
                         + eps * (max(64, v // 256) + 32) * E32 * size)
        p = torch.nan_to_num(torch.exp(torch.where(fin, zd - lse[..., None], -1e30)), 0, 0, 0)
        lse, err = lse[..., None], self.lse_err[..., None]
        q = torch.zeros_like(zd).scatter_(-1, torch.where(y == ignore, 0, y).clamp(0, v - 1)
                                          .long()[..., None], 1 - eps) + eps / v
        self.dz_err = (p * (1 + 2 * zeta * lse.abs()) * (err + (4 * depth + 8) * E32)
                       + 2 * zeta * p * err + 6 * E32 * (p * (1 + 2 * zeta * lse.abs()) + q))
        self.live = y != ignore

    def mean(self):
        n = int(self.live.sum())
        rows = self.loss.numel()
        loss = self.loss.sum() / n
        err = (self.loss_err[self.live].sum() / n
               + (rows / 64 + 20) * E32 * self.loss.abs().sum() / n)
        return loss, err, n

    def grad_bound(self, g, dtype):
        want = self.dz * g
        return want, (self.dz_err + 4 * E32 * self.dz.abs()) * abs(g) \
            + 1.01 * U[dtype] * want.abs() + TINY[dtype]


SHAPES = [(1, 1), (1, 2), (3, 7), (5, 255), (70, 65), (4, 1000), (9, 4096), (7, 4097), (6, 8009),
          (3, 16385), (33, 50257), (2, 65537), (3, 70001), (2, 131077), (3, 150001), (1, 300001)]


def xent_case(n, v, dtype, seed=0, std=2.0, ignored=True):
    z = normal(n, v, std=std, seed=seed).to(dtype)
    y = ids_of((n,), v, seed=seed, kind="flat")
    z.scatter_add_(1, y[:, None], torch.full((n, 1), 4.0).to(dtype))
    if ignored and n > 2:
        y[1::5] = -100
    return z, y


@pytest.mark.parametrize("n,v", SHAPES)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("eps,zeta", [(0.0, 0.0), (0.1, 1e-3)])
def test_cross_entropy(T, n, v, dtype, eps, zeta):
    z, y = xent_case(n, v, dtype)
    c = Xent(z, y, eps, zeta)
    kw = dict(label_smoothing=eps, z_loss=zeta)
    zg, yg = z.to(DEV), y.to(DEV)
    close(T.cross_entropy(zg, yg, reduction="none", **kw), c.loss, c.loss_err)
    loss, err, count = c.mean()
    close(T.cross_entropy(zg, yg, **kw), loss, err)
    close(T.cross_entropy(zg, yg.int(), reduction="sum", **kw), loss * count, err * count)
    # one pass: a mean with a scale, and a sum in place
    got, dz = T.cross_entropy_step(zg, yg, grad_scale=3.0, **kw)
    close(got, loss, err)
    close(dz, *c.grad_bound(3.0 / count, dtype))
    assert torch.equal(zg.cpu(), z)
    work = zg.clone()
    got, dz = T.cross_entropy_step(work, yg, reduction="sum", inplace=True, **kw)
    close(got, loss * count, err * count)
    assert dz.data_ptr() == work.data_ptr()
    close(dz, *c.grad_bound(1.0, dtype))
    # autograd
    leaf = zg.clone().requires_grad_()
    (dz,) = torch.autograd.grad(T.cross_entropy(leaf, yg, **kw) * 2.0, leaf)
    close(dz, *c.grad_bound(2.0 / count, dtype))
    w = torch.rand(n, generator=torch.Generator().manual_seed(2))
    (dz,) = torch.autograd.grad(T.cross_entropy(leaf, yg, reduction="none", **kw), leaf,
                                w.to(DEV))
    want, bound = c.grad_bound(1.0, dtype)
    close(dz, want * w.double()[:, None], bound * w.double()[:, None] + TINY[dtype])


@pytest.mark.parametrize("layout", ["padded", "odd columns", "every other row", "three dims",
                                    "transposed", "shifted", "cut tokens"])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_cross_entropy_of_strided_logits(T, layout, dtype):
    base = normal(6, 20, 1024, dtype=dtype, std=2.0)
    b = base.to(DEV)

    def view(t):
        return {"padded": lambda: t.view(120, 1024)[:, :1000],
                "odd columns": lambda: t.view(120, 1024)[:, 3:704],
                "every other row": lambda: t.view(120, 1024)[::2],
                "three dims": lambda: t[:, :, :999], "transposed": lambda: t.view(120, 1024).T,
                "shifted": lambda: t.view(-1)[1:1 + 100 * 1001].view(100, 1001),
                "cut tokens": lambda: t[:, :-1]}[layout]()
    z = view(base)
    y = ids_of(z.shape[:-1], z.shape[-1], kind="flat")
    c = Xent(z, y)
    loss, err, count = c.mean()
    got, dz = T.cross_entropy_step(view(b), y.to(DEV))
    assert dz.shape == z.shape
    close(got, loss, err)
    close(dz, *c.grad_bound(1.0 / count, dtype))
    leaf = b.clone().requires_grad_()
    (g,) = torch.autograd.grad(T.cross_entropy(view(leaf), y.to(DEV)), leaf)
    close(view(g), *c.grad_bound(1.0 / count, dtype))
    if layout in ("padded", "odd columns", "every other row", "three dims", "shifted"):
        work = b.clone()
        got, dz = T.cross_entropy_step(view(work), y.to(DEV), inplace=True)
        close(view(work), *c.grad_bound(1.0 / count, dtype))
        left = torch.ones(base.shape, dtype=torch.bool)
        view(left).fill_(False)
        assert torch.equal(work.cpu()[left], base[left])   # nothing beside the rows is written


@pytest.mark.parametrize("v", [40, 600, 5000, 50257, 70001, 140001])
def test_masked_and_non_finite_logits(T, v):
    inf, nan = float("inf"), float("nan")
    z, y = xent_case(12, v, F32, ignored=False)
    y[:] = torch.arange(12) + 3
    z[0, 20:] = -inf                 # a mask that leaves a few
    z[1, :] = -inf                   # ... that leaves nothing
    z[2, :] = -inf
    z[2, 5] = 1.5                    # ... the target alone
    z[3, 6] = -inf                   # the target itself masked
    z[4, 30] = nan
    z[5, 30] = inf
    z[6] = torch.finfo(F32).min      # the type's lowest value as a mask, everywhere
    z[7, 1:] = torch.finfo(F32).min
    y[7] = 0
    z[8] = 1e30
    z[9, :] = nan
    y[9] = -100
    z[10, ::2] = -inf
    z[11, 8] = 3e38
    c = Xent(z, y)
    c.loss_err = torch.nan_to_num(c.loss_err, 0.0, 0.0, 0.0)
    assert torch.isnan(c.loss[[1, 4, 5]]).all() and c.loss[3] == inf and c.loss[9] == 0
    zg, yg = z.to(DEV), y.to(DEV)
    close(T.cross_entropy(zg, yg, reduction="none"), c.loss, c.loss_err)
    for got in (T.cross_entropy_step(zg, yg, reduction="sum")[1],
                torch.autograd.grad(T.cross_entropy(zg.requires_grad_(), yg, reduction="sum"),
                                    zg)[0]):
        want, bound = c.grad_bound(1.0, F32)
        live = torch.ones(12, dtype=torch.bool)
        live[[1, 4, 5]] = False      # no softmax
        close(got[live.to(DEV)], want[live], bound[live])
        assert torch.isnan(got[[1, 4, 5]]).all()
        assert not got[9].any()


def test_targets_outside_the_classes(T):
    z, _ = xent_case(6, 50, F32)
    y = torch.tensor([3, -1, 50, 2 ** 40, -100, 49])
    zg = z.to(DEV).requires_grad_()
    loss = T.cross_entropy(zg, y.to(DEV), reduction="none")
    assert torch.isnan(loss).tolist() == [False, True, True, True, False, False]
    dz = torch.autograd.grad(loss.sum(), zg)[0]
    assert torch.isnan(dz).all(1).tolist() == [False, True, True, True, False, False]
    _, dz = T.cross_entropy_step(z.to(DEV), y.to(DEV), reduction="sum")
    assert torch.isnan(dz).all(1).tolist() == [False, True, True, True, False, False]
    assert torch.isfinite(T.cross_entropy(z.to(DEV), y.to(DEV).clamp(0, 49), ignore_index=7))


def test_no_targets(T):
    z, y = xent_case(5, 300, BF16)
    y[:] = 7
    loss, dz = T.cross_entropy_step(z.to(DEV), y.to(DEV), ignore_index=7)
    assert torch.isnan(loss) and not dz.any()
    loss, dz = T.cross_entropy_step(z.to(DEV), y.to(DEV), ignore_index=7, reduction="sum")
    assert loss == 0 and not dz.any()
    none = z.to(DEV)[:0]
    assert torch.isnan(T.cross_entropy(none, y.to(DEV)[:0]))
    assert T.cross_entropy(none, y.to(DEV)[:0], reduction="sum") == 0
    assert T.cross_entropy(none, y.to(DEV)[:0], reduction="none").shape == (0,)
    assert T.cross_entropy_step(none, y.to(DEV)[:0])[1].shape == (0, 300)
    assert T.cross_entropy(z.to(DEV)[0], y.to(DEV)[0]).shape == ()


def test_cross_entropy_gradient_against_differences(T):
    z, y = xent_case(40, 3001, F32)
    d = torch.sign(normal(40, 3001, seed=9))
    kw = dict(label_smoothing=0.1, z_loss=1e-3, reduction="none")
    leaf = z.to(DEV).requires_grad_()
    loss = T.cross_entropy(leaf, y.to(DEV), **kw)
    (dz,) = torch.autograd.grad(loss.sum(), leaf)
    h = 2.0 ** -6
    with torch.no_grad():
        up = T.cross_entropy(leaf + h * d.to(DEV), y.to(DEV), **kw).double()
        down = T.cross_entropy(leaf - h * d.to(DEV), y.to(DEV), **kw).double()
    slope = (dz.double() * d.to(DEV)).sum(1)
    # third derivatives along d: at most 2 of lse, and 6 zeta (|lse| + 1) more of its square;
    # each loss is off by its bound, and z +- h d by half a last place of 16
    c = Xent(z, y, 0.1, 1e-3)
    bound = h * h / 6 * (2 + 6e-3 * 20) + (c.loss_err + 16 * E32) / h \
        + (c.dz_err + 4 * E32 * c.dz.abs()).sum(1)
    close((up - down) / (2 * h), slope.cpu(), bound)


def test_cross_entropy_repeats_its_bits(T):
    z, y = xent_case(3000, 1009, BF16)
    zg, yg = z.to(DEV), y.to(DEV)
    first = T.cross_entropy_step(zg, yg)
    for _ in range(3):
        again = T.cross_entropy_step(zg, yg)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_logits_past_32_bit_offsets(T):
    n, v = 43000, 50257               # 2^31 elements and more
    z = torch.zeros((n, v), dtype=BF16, device=DEV)
    y = torch.zeros(n, dtype=torch.int64, device=DEV)
    z[-1, 9], y[-1] = 12.0, 9
    want = xent_case(1, v, BF16)[0] * 0
    want[0, 9] = 12.0
    c = Xent(want, torch.tensor([9]))
    loss, dz = T.cross_entropy_step(z, y, reduction="sum")
    close(dz[-1:], *c.grad_bound(1.0, BF16))
    close(T.cross_entropy(z[-1:], y[-1:], reduction="none"), c.loss, c.loss_err)
    close(loss / n, (c.loss[0] + (n - 1) * torch.log(torch.tensor(float(v)).double())) / n,
          (n / 64 + 300) * E32 * 11)


def test_cross_entropy_refusals(T, Err):
    z, y = torch.ones(4, 9, device=DEV), torch.zeros(4, dtype=torch.int64, device=DEV)
    for call in (lambda: T.cross_entropy(z.double(), y), lambda: T.cross_entropy(z, y.float()),
                 lambda: T.cross_entropy(z, y[:3]), lambda: T.cross_entropy(z, y.cpu()),
                 lambda: T.cross_entropy(z[:, :0], y), lambda: T.cross_entropy(z[0, 0], y[0]),
                 lambda: T.cross_entropy(z, y, label_smoothing=1.5),
                 lambda: T.cross_entropy(z, y, label_smoothing=-0.1),
                 lambda: T.cross_entropy(z, y, z_loss=-1.0),
                 lambda: T.cross_entropy(z, y, z_loss=float("nan")),
                 lambda: T.cross_entropy(z, y, reduction="max"),
                 lambda: T.cross_entropy_step(z, y, reduction="none"),
                 lambda: T.cross_entropy_step(z.T, torch.zeros_like(y).expand(9, 4)[:, 0],
                                              inplace=True),
                 lambda: T.cross_entropy_step(z[:1].expand(4, 9), y, inplace=True)):
        with pytest.raises(Err):
            call()


# ---- together ---------------------------------------------------------------------------------
def test_on_another_stream(T):
    z, y = xent_case(64, 8009, BF16)
    ids, w = ids_of((8, 100), 500), normal(500, 96)
    side = torch.cuda.Stream()
    zg, yg, ig, wg = z.to(DEV), y.to(DEV), ids.to(DEV), w.to(DEV)

    def all_of():
        x = T.embedding(ig, wg, dropout_p=0.1, rng=RNG)
        return (x, T.dropout(x, 0.3, RNG, residual=x),
                T.embedding_backward(x, ig, 500, pos_rows=100)[0], *T.cross_entropy_step(zg, yg))
    here = all_of()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = all_of()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(here, there):
        assert torch.equal(a, b)


def test_in_a_captured_graph(T):
    """Every replay equals the eager calls on what the inputs hold then, masks included."""
    ids = ids_of((8, 300), 900).to(DEV)
    w, pos = normal(900, 72).to(DEV), normal(300, 72, seed=1).to(DEV)
    z, y = xent_case(100, 3001, BF16)
    z, y = z.to(DEV), y.to(DEV)
    state = torch.tensor([5, 0], device=DEV)

    def step():
        x = T.embedding(ids, w, pos, dropout_p=0.1, rng=state)
        d = T.dropout(x, 0.2, state, residual=x)
        dw, dp = T.embedding_backward(d, ids, 900, pos_rows=300, dropout_p=0.1, rng=state)
        return (x, d, dw, dp, *T.cross_entropy_step(z, y))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for k in range(4):
        state[1] += 1
        ids.copy_(ids_of((8, 300), 900, seed=k))
        z.copy_(xent_case(100, 3001, BF16, seed=k)[0])
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b), k


def test_model_step_matches_torch():
    """The GPT-2 training step of the benchmark with these operators and with torch's, in fp32:
    the same loss and gradients.  Each gradient differs by the rounding of sums of some thousand
    fp32 terms (2^-24 each, relative to its norm) at each of a dozen products on its way."""
    import bench
    tok = ids_of((3, 41), 517, kind="flat").to(DEV)
    got = {}
    for ops in ("torch", "hip"):
        torch.manual_seed(0)
        m = bench._gpt2(517, 64, 64, 2, 4, ops).to(DEV)
        loss = m.train_step(tok[:, :-1], tok[:, 1:], autocast=False)
        got[ops] = float(loss), {n: p.grad for n, p in m.named_parameters()}
    (a, ga), (b, gb) = got["torch"], got["hip"]
    assert abs(a - b) <= 1e-5 * a
    assert ga.keys() == gb.keys()
    for n in ga:
        assert float((ga[n] - gb[n]).norm()) <= 12 * 2000 * E32 * float(ga[n].norm()), n


def test_model_step_with_dropout_follows_the_seed():
    import bench
    tok = ids_of((3, 41), 517, kind="flat").to(DEV)
    m = bench._gpt2(517, 64, 64, 2, 4, "hip", 0.3).to(DEV)
    losses = []
    for seed in (1, 2, 1):
        torch.manual_seed(seed)
        losses.append(float(m.train_step(tok[:, :-1], tok[:, 1:])))
    assert losses[0] == losses[2] != losses[1]
    assert all(torch.isfinite(p.grad).all() for p in m.parameters())


def test_writes_in_place_are_seen_by_autograd(T):
    h, y = normal(64, 96).to(DEV).requires_grad_(), ids_of((64,), 300).to(DEV)
    w = normal(96, 300, seed=1).to(DEV)
    want = torch.autograd.grad(z := h @ w, h, T.cross_entropy_step(z, y)[1])[0]
    z = h @ w
    dz = T.cross_entropy_step(z, y, inplace=True)[1]
    assert torch.equal(torch.autograd.grad(z, h, dz)[0], want)
    z = torch.tanh(h @ w)
    dz = T.cross_entropy_step(z, y, inplace=True)[1]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward(dz)
    dw, g = torch.zeros(300, 96, device=DEV), normal(64, 96).to(DEV)
    before = dw._version
    T.embedding_backward(g, y, 300, weight_grad=dw)
    assert dw._version == before + 1


@pytest.mark.parametrize("v", [200, 1000, 8009, 32003, 150001])
@pytest.mark.parametrize("eps", [0.0, 0.1])
@pytest.mark.parametrize("offset", [0.0, 30.0, -1000.0, 1e4])
def test_what_all_logits_have_in_common_costs_nothing(T, v, eps, offset):
    """Rows that are sure of their target, far from zero.  The bounds know differences of logits
    alone: rho is the relative error of a row's sum (Xent), a loss adds the rounding of its
    three terms and of the logarithm, and the sum of differences that many of the largest."""
    z = normal(24, v, seed=v)
    y = ids_of((24,), v, seed=3, kind="flat")
    z[torch.arange(24), y] += torch.linspace(0.0, 24.0, 24)
    z += offset
    c = Xent(z, y, eps)
    zd = z.double()
    m = zd.amax(1)
    depth = m - zd.amin(1)
    chain = max(64, v // 256) + 32
    rho = (chain + 4 * depth) * E32
    gap = m - zd.gather(1, y[:, None])[:, 0]
    size = torch.log(torch.exp(zd - m[:, None]).sum(1)) + gap + eps * depth
    loss_err = rho + 6 * E32 * size + eps * chain * E32 * depth
    p = torch.exp(zd - torch.logsumexp(zd, 1, keepdim=True))
    q = (c.dz - p).abs()
    dz_err = p * (rho[:, None] + (4 * (m[:, None] - zd) + 8) * E32) + 6 * E32 * (p + q)
    zg, yg = z.to(DEV), y.to(DEV)
    close(T.cross_entropy(zg, yg, label_smoothing=eps, reduction="none"), c.loss, loss_err)
    loss, dz = T.cross_entropy_step(zg, yg, label_smoothing=eps, reduction="sum")
    close(loss, c.loss.sum(), loss_err.sum() + 24 * E32 * c.loss.sum())
    close(dz, c.dz, dz_err)
    leaf = zg.requires_grad_()
    for red, g in (("sum", torch.ones(())), ("none", torch.ones(24))):
        loss = T.cross_entropy(leaf, yg, label_smoothing=eps, reduction=red)
        close(torch.autograd.grad(loss, leaf, g.to(DEV))[0], c.dz, dz_err)


@pytest.mark.parametrize("v", [50, 5000, 150001])
def test_smoothed_losses_of_lowest_and_highest_values(T, v):
    """Masks of the type's lowest value count in the mean over the classes, and no sum of them
    overflows: z times 2^-28 keeps every bit."""
    low = torch.finfo(F32).min
    z, y = xent_case(6, v, F32, ignored=False)
    y[:] = torch.arange(6) + 10
    z[0, 30:] = low
    z[1, y[1]] = low                     # the target itself
    z[2] = low
    z[3, ::2] = low / 4
    z[4, 3:8] = -low / 4
    z[5, 40] = -float("inf")
    want = R.xent(z, y, eps=0.1)[0]
    size = torch.where(torch.isfinite(z), z.double().abs(), 0.0).amax(1)
    got = T.cross_entropy(z.to(DEV), y.to(DEV), label_smoothing=0.1, reduction="none")
    close(got, want, (max(64, v // 256) + 40) * E32 * (2 * size + 20))
    assert want[5] == float("inf") and torch.isfinite(want[:5]).all()


@pytest.mark.parametrize("n,v", [(5, 40), (33, 5001), (3, 200001)])
def test_entries_that_keep_lse(n, v):
    """The C entries whose statistic is lse alone."""
    from defmuon_amd import _native
    lib = _native.load()
    z, y = xent_case(n, v, F32)
    c = Xent(z, y, 0.1, 1e-3)
    zg, yg = z.to(DEV), y.to(DEV)
    loss, lse, ws = (torch.empty(k, device=DEV) for k in (1, n, n))
    count, go, dz = torch.empty(1, device=DEV), torch.ones(1, device=DEV), torch.empty_like(zg)
    stream = torch.cuda.current_stream().cuda_stream
    args = (stream, zg.data_ptr(), 0, n, v, v, yg.data_ptr(), 1, -100, 0.1, 1e-3)
    assert lib.dmh_cross_entropy(*args, 1, 1.0, loss.data_ptr(), count.data_ptr(), lse.data_ptr(),
                                 None, v, ws.data_ptr(), 4 * n) == 0
    assert lib.dmh_cross_entropy_grad(*args, lse.data_ptr(), count.data_ptr(), go.data_ptr(), 0,
                                      dz.data_ptr(), v) == 0
    want, err, live = c.mean()
    close(loss[0], want, err)
    assert int(count) == live
    close(lse, torch.where(c.live, torch.logsumexp(z.double(), 1), 0.0), c.lse_err)
    close(dz, *c.grad_bound(1.0 / live, F32))


@pytest.mark.filterwarnings("ignore::DeprecationWarning")
def test_forward_mode_is_refused(T, Err):
    import torch.autograd.forward_ad as fwd
    x, y = normal(4, 8).to(DEV), torch.zeros(4, dtype=torch.int64, device=DEV)
    with fwd.dual_level():
        d = fwd.make_dual(x, torch.ones_like(x))
        for call in (lambda: T.dropout(d, 0.1, RNG), lambda: T.dropout(x, 0.1, RNG, residual=d),
                     lambda: T.embedding(y, d), lambda: T.embedding(y, x, d, positions=y),
                     lambda: T.embedding_backward(x, y, 4, weight_grad=d),
                     lambda: T.cross_entropy(d, y), lambda: T.cross_entropy_step(d, y)):
            with pytest.raises(Err, match="forward-mode"):
                call()
        T.dropout(x, 0.1, RNG, residual=x)   # no tangent, no refusal


@pytest.mark.filterwarnings("ignore")
def test_traces(T, Err):
    from torch.fx.experimental.proxy_tensor import make_fx
    w, w2 = normal(50, 24).to(DEV), normal(50, 24, seed=1).to(DEV)
    ids, y = ids_of((9,), 50).to(DEV), ids_of((9,), 24).to(DEV)

    def step(t):
        x = T.embedding(ids, t, dropout_p=0.1, rng=RNG)
        return T.cross_entropy(T.dropout(x, 0.2, RNG, residual=x), y)
    for grad in (False, True):
        traced = torch.jit.trace(step, w.clone().requires_grad_(grad))
        assert torch.equal(traced(w2), step(w2))
    for call in (step, lambda t: T.dropout_backward(t, 0.1, RNG),
                 lambda t: T.cross_entropy_step(t[:9], y)[1]):
        with pytest.raises(Err, match="trace"):
            make_fx(call)(w)


@pytest.mark.parametrize("dim", [9, 15, 500, 513, 519, 1025, 1027, 2049])
@pytest.mark.parametrize("tokens,rows", [(200, 300), (3000, 40), (9000, 700)])
@pytest.mark.parametrize("out", [F32, BF16])
def test_overlapping_columns_are_added_once(T, dim, tokens, rows, out):
    """Widths whose last eight columns share some with the piece before, in the same wave and
    (8 x 64 n + 1 .. 7) in another: each sum is added once, in one launch, chunk by chunk and
    joined, for the sums of either table."""
    ids, t = ids_of((tokens,), rows), ids_of((tokens,), 64, seed=1)
    g = normal(tokens, dim)
    w0, p0 = normal(rows, dim, dtype=out, seed=5), normal(64, dim, dtype=out, seed=6)
    w, pg = w0.to(DEV), p0.to(DEV)
    for _ in range(2):
        T.embedding_backward(g.to(DEV), ids.to(DEV), rows, pos_rows=64, positions=t.to(DEV),
                             weight_grad=w, pos_grad=pg)
        for got, first, idx in ((w, w0, ids), (pg, p0, t)):
            want, size, n = R.table_grad(g, idx, first.shape[0])
            want = want + first.double()
            close(got, want, grad_bound(want, size + first.double().abs(), n, out))
        w0, p0 = w.cpu(), pg.cpu()


def test_positions_of_another_type_outside_the_table(T):
    w, pos = normal(10, 24).to(DEV), normal(4, 24, seed=1).to(DEV)
    ids, t = torch.tensor([3, 1, 4, 9, 2]), torch.tensor([1, 2 ** 32 + 1, -2 ** 32, 2 ** 31, 3])
    g = normal(5, 24)
    for i, p in ((ids.int(), t), (t, ids.int() % 4)):
        y = T.embedding(i.to(DEV), w, pos, positions=p.to(DEV)).cpu()
        ok = (i >= 0) & (i < 10) & (p >= 0) & (p < 4)
        assert torch.equal(torch.isnan(y).all(1), ~ok) and not torch.isnan(y[ok]).any()
        dw, dp = T.embedding_backward(g.to(DEV), i.to(DEV), 10, pos_rows=4, positions=p.to(DEV))
        for got, idx, rows in ((dw, i, 10), (dp, p, 4)):
            want, size, n = R.table_grad(g, idx, rows)
            close(got, want, grad_bound(want, size, n, F32))


def test_a_position_table_without_rows(T):
    """Every position is outside it."""
    w, none = normal(10, 24).to(DEV).requires_grad_(), torch.empty(0, 24, device=DEV)
    ids = torch.tensor([3, 1, 4]).to(DEV)
    y = T.embedding(ids, w, none, positions=torch.zeros_like(ids))
    assert torch.isnan(y).all()
    g = normal(3, 24)
    (dw,) = torch.autograd.grad(y, w, g.to(DEV))
    want, size, n = R.table_grad(g, ids.cpu(), 10)
    close(dw, want, grad_bound(want, size, n, F32))
    assert torch.isnan(T.embedding(ids, none, none, positions=ids)).all()
    assert torch.isnan(T.embedding(ids, none)).all()
    assert T.embedding(ids[:0], w, none).shape == (0, 24)
    # no rows, no gradient of them
    assert T.embedding_backward(g.to(DEV), ids, 10, pos_rows=0, positions=ids)[1] is None


@pytest.mark.parametrize("dim", [1, 2, 3, 4, 5, 6, 7])
@pytest.mark.parametrize("kind", ["same", "zipf"])
@pytest.mark.parametrize("dtype,out,p", [(F32, F32, 0.0), (BF16, BF16, 0.2)])
def test_narrow_tables_of_many_tokens(T, dim, kind, dtype, out, p):
    """Terms of one sign, one id for most of 200000 tokens.  No sum adds more in sequence than a
    chunk's 32, one in 32 of the chunks, 32 of those and the first chunk's, and two roundings
    each of the scales and the sum."""
    n, rows = 200000, 50
    ids = ids_of((n,), rows, kind=kind)
    g = (normal(n, dim).abs() * 0.01 + 0.1).to(dtype)
    kw = dict(scale=1.5, dropout_p=p, rng=RNG)
    dw, dp = T.embedding_backward(g.view(2000, 100, dim).to(DEV), ids.view(2000, 100).to(DEV),
                                  rows, pos_rows=120, dtype=out, **kw)
    chain = 32 + n / 32 / 32 + 32 + 1 + 4
    want, size, _ = R.table_grad(g, ids, rows, 1.5, p, RNG)
    close(dw, want, chain * E32 * size + 1.01 * U[out] * want + TINY[out])
    t = torch.arange(100).repeat(2000)
    want, size, _ = R.table_grad(g, t, 120, 1.0, p, RNG)
    close(dp, want, chain * E32 * size + 1.01 * U[out] * want + TINY[out])
    # added to what a table holds, its other rows untouched
    w0 = normal(rows + 70, dim, dtype=out)
    w = w0.to(DEV)
    T.embedding_backward(g.to(DEV), ids.to(DEV), rows + 70, weight_grad=w, **kw)
    want, size, terms = R.table_grad(g, ids, rows + 70, 1.5, p, RNG)
    total = want + w0.double()
    close(w, total, chain * E32 * size + 1.01 * U[out] * total.abs() + E32 * w0.double().abs()
          + TINY[out])
    gone = terms[:, 0] == 0
    assert gone.any() and torch.equal(w.cpu()[gone], w0[gone])


def test_more_tokens_of_one_id_than_fp32_counts(T):
    """Ones: every sum below 2^24 is exact, and two roundings remain."""
    n = (1 << 24) + 12345
    ids = torch.ones(n, dtype=torch.int32, device=DEV)
    ids[-5:] = 2
    dw, _ = T.embedding_backward(torch.ones(n, 1, device=DEV), ids, 4)
    assert dw[0] == 0 and dw[2] == 5 and dw[3] == 0
    assert abs(float(dw[1]) - (n - 5)) <= 33 * E32 * n


def test_dropout_module_in_a_captured_graph(T, Err):
    """Two layers whose rng are rows of one tensor: the masks differ from each other and from
    replay to replay, and are those of eager calls, gradients too."""
    layers = [T.Dropout(0.4), T.Dropout(0.4)]
    x = normal(64, 96).to(DEV).requires_grad_()
    state = torch.tensor([[7, 0], [7, 1]], device=DEV)

    def step():
        h = layers[0](x, rng=state[0])
        y = layers[1](h, residual=h, rng=state[1])
        return h, y, torch.autograd.grad(y, x, torch.ones_like(y))[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        refused = 0
        for call in (T.draw_rng, lambda: layers[0](x)):
            try:
                call()
            except Err:
                refused += 1
        outs = step()
    assert refused == 2
    before = None
    for k in range(4):
        state[:, 0] += 1
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b), k
        masks = outs[0] != 0, (outs[1] - outs[0]) != 0
        assert not torch.equal(*masks)
        assert before is None or not torch.equal(before, masks[0])
        before = masks[0]


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("grad", [False, True])
def test_compiled_programs_run_the_calls(T, grad):
    """Outside the compiled graphs, as they are: masks drawn at each call among them."""
    w, w2 = normal(50, 24).to(DEV).requires_grad_(grad), normal(24, 24, seed=1).to(DEV)
    ids, y = ids_of((9,), 50).to(DEV), ids_of((9,), 24).to(DEV)
    drop = T.Dropout(0.5)

    def step(t):
        x = T.embedding(ids, t, dropout_p=0.1, rng=RNG) @ w2
        return T.cross_entropy(drop(x * 2, residual=x), y, reduction="none")
    compiled = torch.compile(step, backend="aot_eager")
    runs = []
    for f in (step, compiled, compiled):
        torch.manual_seed(len(runs) // 2)   # the same, the same, another
        loss = f(w)
        runs.append((loss, torch.autograd.grad(loss.sum(), w)[0] if grad else loss))
    for a, b in zip(runs[0], runs[1]):
        assert torch.equal(a, b)
    assert not torch.equal(runs[1][0], runs[2][0])
    torch._dynamo.reset()


def test_in_place_gradients_of_views(T):
    """From the view, and from the product's own output: the same gradient."""
    h, y = normal(6, 10, 96).to(DEV).requires_grad_(), ids_of((60,), 304, kind="flat").to(DEV)
    w = normal(96, 304, seed=1).to(DEV)
    want = torch.autograd.grad(z := h @ w, h, T.cross_entropy_step(z.view(-1, 304), y)[1]
                               .view_as(z))[0]
    z = h @ w
    dz = T.cross_entropy_step(z.view(-1, 304), y, inplace=True)[1]
    assert dz.data_ptr() == z.data_ptr()
    assert torch.equal(torch.autograd.grad(z, h, dz.view_as(z))[0], want)
    view = (h @ w).view(-1, 304)
    dz = T.cross_entropy_step(view, y, inplace=True)[1]
    assert torch.equal(torch.autograd.grad(view, h, dz)[0], want)
