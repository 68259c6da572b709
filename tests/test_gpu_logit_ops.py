"""Log probabilities, entropies, top classes and distillation on the GPU against their plain forms
in 64 bits (bounds: logit_ref)."""

import pytest
import torch

import logit_ref as L
from train_ref import E32, TINY, close

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


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


def gpu(t):
    return None if t is None else t.to(DEV)


SHAPES = [(1, 1), (1, 2), (3, 7), (5, 255), (70, 65), (4, 1000), (9, 4096), (7, 4097), (6, 8009),
          (3, 8193), (3, 16385), (2, 32771), (33, 50257), (2, 65537), (3, 70001), (2, 131077),
          (2, 150001), (1, 300001)]


def lp_case(n, v, dtype, seed=0, std=2.0):
    z = normal(n, v, std=std, seed=seed).to(dtype)
    y = torch.randint(0, v, (n,), generator=torch.Generator().manual_seed(seed))
    z.scatter_add_(1, y[:, None], torch.full((n, 1), 4.0).to(dtype))
    if n > 2:
        y[1::5] = -100
    return z, y


def check_log_probs(got, z, y, k, tau, what=""):
    want, ids = L.log_probs(z, y, k, tau)
    for name, (value, bound) in want.items():
        close(getattr(got, name), value, torch.nan_to_num(bound, 0.0, 0.0, 0.0), (what, name))
    if k:
        rows = torch.isfinite(L.Softmax(z).lse[..., 0])
        assert torch.equal(got.top_ids.cpu()[rows], ids[rows]), what
    assert (got.log_probs is None) == (y is None) and (got.top_ids is None) == (k == 0)


# ---- log probabilities ------------------------------------------------------------------------
@pytest.mark.parametrize("n,v", SHAPES)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("tau,k", [(1.0, 0), (0.7, 5), (2.0, 64)])
def test_log_probs(T, n, v, dtype, tau, k):
    z, y = lp_case(n, v, dtype)
    k = min(k, v)
    zg, yg = z.to(DEV), y.to(DEV)
    got = T.token_log_probs(zg, yg, top=k, temperature=tau)
    check_log_probs(got, z, y, k, tau)
    again = T.token_log_probs(zg, yg.int(), top=k, temperature=tau)
    for a, b in zip(got, again):
        assert a is None or torch.equal(a, b)
    check_log_probs(T.token_log_probs(zg, top=k, temperature=tau), z, None, k, tau)
    assert torch.equal(zg.cpu(), z)
    # the gradient of all outputs, and of each alone
    gy, gh, gt = normal(n, seed=3), normal(n, seed=4), normal(n, k, seed=5)
    leaf = zg.clone().requires_grad_()
    out = T.token_log_probs(leaf, yg, top=k, temperature=tau)
    ids = None if out.top_ids is None else out.top_ids.cpu()
    for a, b, c in ((gy, gh, gt if k else None), (gy, None, None), (None, gh, None),
                    (None, None, gt if k else None)):
        pairs = [(o, g.to(DEV)) for o, g in zip(out, (a, b, c)) if g is not None]
        if pairs:
            (dz,) = torch.autograd.grad([o for o, _ in pairs], leaf, [g for _, g in pairs],
                                        retain_graph=True)
            assert dz.dtype == dtype
            close(dz, *L.log_probs_grad(z, y, ids, a, b, c, tau, dtype))


def views(base, layout):
    return {"padded": lambda t: t.view(120, 1024)[:, :1000],
            "odd columns": lambda t: t.view(120, 1024)[:, 3:704],
            "every other row": lambda t: t.view(120, 1024)[::2],
            "three dims": lambda t: t[:, :, :999], "transposed": lambda t: t.view(120, 1024).T,
            "shifted": lambda t: t.view(-1)[1:1 + 100 * 1001].view(100, 1001),
            "cut tokens": lambda t: t[:, :-1],
            "one row": lambda t: t[2, 3]}[layout](base)


LAYOUTS = ["padded", "odd columns", "every other row", "three dims", "transposed", "shifted",
           "cut tokens", "one row"]


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_log_probs_of_strided_logits(T, layout, dtype):
    base = normal(6, 20, 1024, dtype=dtype, std=2.0)
    b = base.to(DEV).requires_grad_()
    z = views(base, layout)
    y = torch.randint(0, z.shape[-1], z.shape[:-1], generator=torch.Generator().manual_seed(0))
    out = T.token_log_probs(views(b, layout), y.to(DEV), top=9)
    check_log_probs(out, z, y, 9, 1.0)
    gh, gt = normal(*z.shape[:-1], seed=1), normal(*z.shape[:-1], 9, seed=2)
    (g,) = torch.autograd.grad([out.entropy, out.top_log_probs], b, [gh.to(DEV), gt.to(DEV)])
    close(views(g, layout), *L.log_probs_grad(z, y, out.top_ids.cpu(), None, gh, gt, 1.0, dtype))
    rest = torch.ones(base.shape, dtype=torch.bool)
    views(rest, layout).fill_(False)
    assert not g.cpu()[rest].any()
    # tokens and their gradient in other orders
    if z.ndim == 3:
        yt = y.t().contiguous().t().to(DEV)
        assert torch.equal(T.token_log_probs(views(b, layout), yt).log_probs, out.log_probs)


@pytest.mark.parametrize("v", [40, 600, 5000, 9001, 50257, 70001, 140001])
def test_masked_and_non_finite_logits(T, v):
    inf, nan = float("inf"), float("nan")
    z, _ = lp_case(13, v, F32)
    y = torch.arange(13) + 3
    z[0, 20:] = -inf                 # a mask that leaves a few
    z[1, :] = -inf                   # ... that leaves nothing
    z[2, :] = -inf
    z[2, 5] = 1.5                    # ... the token alone
    z[3, 6] = -inf                   # the token itself masked
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
    z[12, 15:] = -1e4
    out, ids = L.log_probs(z, y, 30)
    zg = z.to(DEV).requires_grad_()
    got = T.token_log_probs(zg, y.to(DEV), top=30)
    bad = torch.tensor([r in (1, 4, 5) for r in range(13)])
    for name, (value, bound) in out.items():
        x = getattr(got, name).cpu()
        close(x[~bad], value[~bad], torch.nan_to_num(bound, 0.0, 0.0, 0.0)[~bad], name)
        assert torch.isnan(x[bad]).all(), name
    assert torch.equal(got.top_ids.cpu()[~bad], ids[~bad])
    assert torch.equal(got.top_ids.cpu()[bad], torch.arange(30).expand(3, 30))
    gy, gh = normal(13, seed=1), normal(13, seed=2)
    (dz,) = torch.autograd.grad([got.log_probs, got.entropy], zg, [gy.to(DEV), gh.to(DEV)])
    dz = dz.cpu()
    want, bound = L.log_probs_grad(z, y, None, gy, gh, None, 1.0, F32)
    ok = ~bad
    close(dz[ok], torch.nan_to_num(want, 0.0, 0.0, 0.0)[ok], bound[ok].nan_to_num(0.0, 0.0, 0.0))
    assert torch.isnan(dz[bad]).all() and not dz[9].any()


def test_tokens_outside_the_classes(T):
    z, _ = lp_case(6, 50, F32)
    y = torch.tensor([3, -1, 50, 2 ** 40, -100, 49])
    zg = z.to(DEV).requires_grad_()
    out = T.token_log_probs(zg, y.to(DEV), top=2)
    bad = [False, True, True, True, False, False]
    assert torch.isnan(out.log_probs).tolist() == bad
    assert torch.isfinite(out.entropy).all() and torch.isfinite(out.top_log_probs).all()
    assert out.top_ids[4].tolist() == [-100, -100] and not out.top_log_probs[4].any()
    (dz,) = torch.autograd.grad(out.log_probs.sum(), zg)
    assert torch.isnan(dz).all(1).tolist() == bad and torch.isfinite(dz[[0, 4, 5]]).all()
    got = T.token_log_probs(zg, y.to(DEV).clamp(0, 49), ignore_index=7)
    assert torch.isfinite(got.log_probs).all()


def test_no_rows(T):
    z = normal(0, 30).to(DEV).requires_grad_()
    y = torch.zeros(0, dtype=torch.int64, device=DEV)
    out = T.token_log_probs(z, y, top=3)
    assert [tuple(o.shape) for o in out] == [(0,), (0,), (0, 3), (0, 3)]
    (dz,) = torch.autograd.grad(out.entropy.sum(), z)
    assert dz.shape == (0, 30)
    ids, t = torch.zeros(0, 2, dtype=torch.int64, device=DEV), torch.zeros(0, 2, device=DEV)
    assert torch.isnan(T.distillation(z, ids, t))
    assert T.distillation(z, ids, t, reduction="sum") == 0
    assert T.distillation(z, ids, t, reduction="none").shape == (0,)
    assert T.distillation_step(z, ids, t)[1].shape == (0, 30)


def rows_of_all_kinds(v, dtype):
    """Rows that select badly: equal, in order, few values, lumps in one place."""
    g = torch.Generator().manual_seed(v)
    z = torch.empty(14, v)
    z[0] = 0.0
    z[1] = -3.0
    z[2] = torch.arange(v) / v
    z[3] = -torch.arange(v) / v
    z[4] = torch.randint(0, 3, (v,), generator=g).float()
    z[5] = torch.randint(-2, 1, (v,), generator=g).float()
    z[6] = torch.zeros(v) * -1.0            # -0 and 0 are equal
    z[6, ::3] = 0.0
    z[7] = torch.randn(v, generator=g)
    z[7, :min(v, 700)] += 20.0              # many large ones side by side
    z[8] = torch.randn(v, generator=g)
    z[8, -min(v, 700):] += 20.0
    z[9] = -float("inf")
    z[9, v // 2] = 1.0
    z[10] = torch.finfo(dtype).min
    z[11] = torch.randn(v, generator=g) * 1e-30
    z[12] = torch.randn(v, generator=g)
    z[12, ::max(1, v // 100)] = 9.0
    z[13] = torch.randn(v, generator=g) - 50.0
    z[13, ::8] += 30.0
    return z.to(dtype)


@pytest.mark.parametrize("v", [3, 64, 300, 1025, 4000, 8192, 9003, 16400, 32768, 50257, 66000,
                               100003, 200003])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_top_classes_of_any_row(T, v, dtype):
    z = rows_of_all_kinds(v, dtype)
    for k in (1, 2, 37, 64, 65, 200, 256):
        if k <= v:
            got = T.token_log_probs(z.to(DEV), top=k)
            assert torch.equal(got.top_ids.cpu(), L.top(z, k)), k
            check_log_probs(got, z, None, k, 1.0, k)


def test_top_of_many_rows_repeats_its_bits(T):
    z = normal(3000, 1009, dtype=BF16).to(DEV)
    first = T.token_log_probs(z, top=50)
    assert torch.equal(first.top_ids.cpu(), L.top(z.cpu(), 50))
    for _ in range(3):
        again = T.token_log_probs(z, top=50)
        assert all(torch.equal(a, b) for a, b in zip(first[1:], again[1:]))


@pytest.mark.parametrize("v", [200, 8009, 50257, 150001])
@pytest.mark.parametrize("offset", [0.0, -1000.0, 1e4])
def test_what_all_logits_have_in_common_costs_nothing(T, v, offset):
    """The bounds know differences of logits alone."""
    z = normal(24, v, seed=v)
    y = torch.randint(0, v, (24,), generator=torch.Generator().manual_seed(3))
    z[torch.arange(24), y] += torch.linspace(0.0, 24.0, 24)
    z += offset
    check_log_probs(T.token_log_probs(z.to(DEV), y.to(DEV), top=4), z, y, 4, 1.0)


def test_log_prob_gradient_against_differences(T):
    z, y = lp_case(40, 3001, F32)
    d = torch.sign(normal(40, 3001, seed=9))
    leaf = z.to(DEV).requires_grad_()
    gy, gh = normal(40, seed=1).to(DEV), normal(40, seed=2).to(DEV)

    def f(t):
        out = T.token_log_probs(t, y.to(DEV), temperature=1.5)
        return out.log_probs.double() * gy + out.entropy.double() * gh
    (dz,) = torch.autograd.grad(f(leaf).sum(), leaf)
    h = 2.0 ** -6
    with torch.no_grad():
        up, down = f(leaf + h * d.to(DEV)), f(leaf - h * d.to(DEV))
    slope = (dz.double() * d.to(DEV)).sum(1)
    # along d, |d| <= 1 / tau: third derivatives of lse at most 2, of the entropy (through E[x]
    # and its covariances with d) at most 24 (1 + H + max gap)
    want, _ = L.log_probs(z, y, 0, 1.5)
    s = L.Softmax(z, 1.5)
    third = 2 * gy.cpu().abs() + 24 * gh.cpu().abs() * (1 + s.h + s.gap.amax(1, True))[:, 0]
    err = (want["log_probs"][1] + 16 * E32) * gy.cpu().abs() \
        + (want["entropy"][1] + 32 * E32) * gh.cpu().abs()
    _, bound = L.log_probs_grad(z, y, None, gy.cpu(), gh.cpu(), None, 1.5, F32)
    close((up - down) / (2 * h), slope.cpu(), h * h / 6 * third + err / h + bound.sum(1))


def test_log_probs_past_32_bit_offsets(T):
    n, v = 43000, 50257               # 2^31 elements and more
    z = torch.zeros((n, v), dtype=BF16, device=DEV)
    z[-1, 9], z[-1, 50256] = 12.0, 11.0
    y = torch.full((n,), 9, device=DEV)
    want = torch.zeros(1, v, dtype=BF16)
    want[0, 9], want[0, 50256] = 12.0, 11.0
    leaf = z.requires_grad_()
    out = T.token_log_probs(leaf, y, top=3)
    ref, ids = L.log_probs(want, torch.tensor([9]), 3)
    assert out.top_ids[-1].tolist() == ids[0].tolist() == [9, 50256, 0]
    assert out.top_ids[0].tolist() == [0, 1, 2]
    close(out.log_probs[-1:], *ref["log_probs"])
    (dz,) = torch.autograd.grad(out.log_probs[-1], leaf)
    close(dz[-1:], *L.log_probs_grad(want, torch.tensor([9]), None, torch.ones(1), None, None, 1.0,
                                     BF16))


def test_log_prob_refusals(T, Err):
    z, y = torch.ones(4, 9, device=DEV), torch.zeros(4, dtype=torch.int64, device=DEV)
    for call in (lambda: T.token_log_probs(z.double(), y), lambda: T.token_log_probs(z, y.float()),
                 lambda: T.token_log_probs(z, y.cpu()), lambda: T.token_log_probs(z, y[:3]),
                 lambda: T.token_log_probs(z, top=10), lambda: T.token_log_probs(z, top=-1),
                 lambda: T.token_log_probs(z, temperature=0.0),
                 lambda: T.token_log_probs(z, temperature=float("inf"))):
        with pytest.raises(Err):
            call()


# ---- distillation -----------------------------------------------------------------------------
def kd_case(n, v, k, dtype=F32, teacher=F32, seed=0, ragged=True, cover=0.9):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(n, v, generator=g) * 2).to(dtype)
    ids = torch.stack([torch.randperm(v, generator=g)[:k] for _ in range(n)])
    t = torch.log_softmax(torch.randn(n, k, generator=g) * 2, 1) + torch.log(torch.tensor(cover))
    z.scatter_add_(1, ids, (t + 7.0 + torch.randn(n, k, generator=g)).to(dtype))
    if n > 2:
        ids[1::5] = -100                    # no teacher
        if ragged and k > 2:
            ids[2::4, -1] = -100            # a shorter list
            ids[0, k // 2] = -100           # ... with a gap
    return z, ids, t.to(teacher)


def check_distill(T, z, ids, t, tau, rest, dtype, what=""):
    c = L.Distill(z, ids, t, tau, rest)
    zg, ig, tg = z.to(DEV), ids.to(DEV), t.to(DEV)
    kw = dict(temperature=tau, rest=rest)
    close(T.distillation(zg, ig, tg, reduction="none", **kw), c.loss, c.loss_err, (what, "none"))
    loss, err, count = c.mean()
    close(T.distillation(zg, ig, tg, **kw), loss, err, (what, "mean"))
    close(T.distillation(zg, ig.int(), tg, reduction="sum", **kw), loss * count, err * count)
    got, dz = T.distillation_step(zg, ig, tg, grad_scale=3.0, **kw)
    close(got, loss, err, (what, "step"))
    close(dz, *c.grad_bound(3.0 / count, dtype), (what, "step dz"))
    assert torch.equal(zg.cpu(), z)
    work = zg.clone()
    got, dz = T.distillation_step(work, ig, tg, reduction="sum", inplace=True, **kw)
    close(got, loss * count, err * count)
    assert dz.data_ptr() == work.data_ptr()
    close(dz, *c.grad_bound(1.0, dtype), (what, "in place"))
    leaf = zg.clone().requires_grad_()
    (dz,) = torch.autograd.grad(T.distillation(leaf, ig, tg, **kw) * 2.0, leaf)
    close(dz, *c.grad_bound(2.0 / count, dtype), (what, "autograd"))
    w = torch.rand(z.shape[0], generator=torch.Generator().manual_seed(2))
    (dz,) = torch.autograd.grad(T.distillation(leaf, ig, tg, reduction="none", **kw), leaf,
                                w.to(DEV))
    want, bound = c.grad_bound(1.0, dtype)
    w = w.double()[:, None]
    close(dz, want * w, bound * w + 4 * E32 * want.abs() * w + TINY[dtype], (what, "rows"))


@pytest.mark.parametrize("n,v", [s for s in SHAPES if s[1] >= 7])
@pytest.mark.parametrize("dtype,teacher", [(F32, F32), (BF16, F32), (F16, BF16)])
@pytest.mark.parametrize("tau,rest,k", [(1.0, False, 16), (2.0, True, 5), (0.7, True, 70)])
def test_distillation(T, n, v, dtype, teacher, tau, rest, k):
    k = min(k, v // 2)
    z, ids, t = kd_case(n, v, k, dtype, teacher)
    check_distill(T, z, ids, t, tau, rest, dtype)


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("v,k", [(2000, 257), (9000, 1024), (60000, 1000), (1024, 1024), (5, 5),
                                 (1, 1), (2, 1), (140001, 600)])
def test_long_lists(T, v, k, rest):
    z, ids, t = kd_case(3, v, k, cover=0.8)
    if rest and k == v:                     # nothing beside the list: all of the teacher on it
        t = torch.log_softmax(t.double(), 1).float() + 1e-3
    check_distill(T, z, ids, t, 1.3, rest, F32)


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("v", [50, 9001, 70001, 140001])
def test_classes_listed_twice(T, v, rest):
    z, ids, t = kd_case(6, v, 20, cover=0.7, ragged=False)
    ids[0, 1] = ids[0, 0]
    ids[2] = ids[2, 0]                      # one class alone
    ids[3, 10:] = ids[3, :10].flip(0)
    check_distill(T, z, ids, t, 1.0, rest, F32)
    zg, ig, tg = z.to(DEV), ids.to(DEV), t.to(DEV)
    first = T.distillation_step(zg, ig, tg, rest=rest)
    for _ in range(3):
        again = T.distillation_step(zg, ig, tg, rest=rest)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_distillation_of_strided_logits(T, layout, dtype):
    base = normal(6, 20, 1024, dtype=dtype, std=2.0)
    b, z = base.to(DEV), views(base, layout)
    g = torch.Generator().manual_seed(1)
    k, v = 12, z.shape[-1]
    ids = torch.rand(*z.shape[:-1], v, generator=g).argsort(-1)[..., :k]
    t = torch.log_softmax(torch.randn(*ids.shape, generator=g), -1) - 0.2
    c = L.Distill(z, ids, t, 1.0, True)
    loss, err, count = c.mean()
    # lists whose memory has another order
    ig = ids.to(DEV).transpose(-1, 0).contiguous().transpose(-1, 0)
    tg = torch.stack([t, t], -1).to(DEV)[..., 0]
    got, dz = T.distillation_step(views(b, layout), ig, tg, rest=True)
    assert dz.shape == z.shape
    close(got, loss, err)
    close(dz, *c.grad_bound(1.0 / count, dtype))
    leaf = b.clone().requires_grad_()
    (gz,) = torch.autograd.grad(T.distillation(views(leaf, layout), ig, tg, rest=True), leaf)
    close(views(gz, layout), *c.grad_bound(1.0 / count, dtype))
    if layout not in ("transposed", "cut tokens"):
        work = b.clone()
        T.distillation_step(views(work, layout), ig, tg, rest=True, inplace=True)
        close(views(work, layout), *c.grad_bound(1.0 / count, dtype))
        left = torch.ones(base.shape, dtype=torch.bool)
        views(left, layout).fill_(False)
        assert torch.equal(work.cpu()[left], base[left])   # nothing beside the rows is written


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("v", [60, 600, 9001, 50257, 70001, 140001])
def test_masked_and_non_finite_rows(T, v, rest):
    inf, nan = float("inf"), float("nan")
    z, ids, t = kd_case(16, v, 8, ragged=False)
    ids[:] = torch.arange(8) * 6 + 1
    z[0, 43:] = -inf                     # the rest partly masked
    z[1] = -inf                          # no softmax
    z[2, 30] = nan
    z[3, 40] = inf
    z[4, 1] = -inf                       # a listed class masked: infinitely far
    z[5, 1] = -inf
    t[5, 0] = -inf                       # ... of which the teacher has nothing
    t[6, 3] = nan
    ids[7, 2] = v                        # outside
    ids[8, 7] = -1
    ids[9, 0] = -100
    z[9] = nan                           # no teacher: never read
    t[9] = nan
    z[10] = torch.finfo(F32).min
    t[11] += 5.0                         # sums to more than 1
    z[12, 7:] -= 200.0                   # a student without a doubt, of one class of the list
    z[13] += 1000.0
    t[14] = -inf                         # the teacher has nothing on the list
    z[15] = -inf
    z[15, :44] = 1.0
    c = L.Distill(z, ids, t, 1.0, rest)
    nans = torch.isnan(c.loss)
    assert nans.tolist() == [r in (1, 2, 3, 6, 7, 8) or (r == 14 and not rest) for r in range(16)]
    assert c.loss[4] == inf and torch.isfinite(c.loss[[5, 12]]).all() and c.loss[9] == 0
    zg, ig, tg = z.to(DEV), ids.to(DEV), t.to(DEV)
    close(T.distillation(zg, ig, tg, rest=rest, reduction="none"), c.loss, c.loss_err)
    want, bound = c.grad_bound(1.0, F32)
    leaf = zg.clone().requires_grad_()
    for dz in (T.distillation_step(zg, ig, tg, rest=rest, reduction="sum")[1],
               torch.autograd.grad(T.distillation(leaf, ig, tg, rest=rest, reduction="sum"),
                                   leaf)[0]):
        dz = dz.cpu()
        close(dz[~nans], want[~nans], bound[~nans])
        assert torch.isnan(dz[nans]).all() and not dz[9].any()


@pytest.mark.parametrize("v", [24, 600, 9001, 50257, 140001])
def test_no_class_beside_the_list(T, v):
    """A mask that leaves 20 classes to both, or a list of all: what rounding leaves of the
    teacher's 1 belongs to no class and does not count."""
    k, inf = 24, float("inf")
    teacher, student = normal(40, v, std=3.0), normal(40, v, seed=1)
    teacher[:30, v // 2 + 10:] = student[:30, v // 2 + 10:] = -inf
    teacher[:30, :v // 2 - 10] = student[:30, :v // 2 - 10] = -inf
    out = T.token_log_probs(teacher.to(DEV), top=k, temperature=1.5)
    ids, t = out.top_ids.cpu(), out.top_log_probs.cpu()
    assert (torch.exp(t[:30].double()).sum(1) < 1).any() and (t[:30, 20:] == -inf).all()
    t[29] = -inf                         # ... and nothing on the list: no distribution at all
    t[28] -= 1.0                         # less than 1 by far
    c = L.Distill(student, ids, t, 1.5, True)
    nans = torch.isnan(c.loss)
    assert nans.nonzero().tolist() == [[29]] and torch.isfinite(c.loss[~nans]).all()
    sg, ig, tg = student.to(DEV), ids.to(DEV), t.to(DEV)
    kw = dict(temperature=1.5, rest=True)
    close(T.distillation(sg, ig, tg, reduction="none", **kw), c.loss, c.loss_err)
    want, bound = c.grad_bound(1.0, F32)
    leaf = sg.clone().requires_grad_()
    for dz in (T.distillation_step(sg, ig, tg, reduction="sum", **kw)[1],
               torch.autograd.grad(T.distillation(leaf, ig, tg, reduction="sum", **kw), leaf)[0]):
        dz = dz.cpu()
        close(dz[~nans], want[~nans], bound[~nans])
        assert torch.isnan(dz[nans]).all()


@pytest.mark.parametrize("mask", [-1e9, -1e4, torch.finfo(F32).min])
@pytest.mark.parametrize("v", [600, 9001, 50257, 140001])
def test_masks_beside_the_list(T, v, mask):
    """Masks of finite values: what the rounding of the teacher's list leaves of its 1 is far from
    the masked classes, but is none of theirs: the same as with masks of -inf."""
    k, n = 24, 60
    teacher, student = normal(n, v, std=3.0), normal(n, v, seed=1)
    hidden = torch.ones(v, dtype=torch.bool)
    hidden[v // 2:v // 2 + 20] = False
    teacher[:, hidden] = student[:, hidden] = mask
    out = T.token_log_probs(teacher.to(DEV), top=k)
    ids, t = out.top_ids.cpu(), out.top_log_probs.cpu()
    left = 1 - torch.exp(t.double()).sum(1)
    assert (left > 0).any() and left.max() < 8 * L.E32
    c = L.Distill(student.masked_fill(hidden, -float("inf")), ids,
                  t.masked_fill(t < mask / 2, -float("inf")), 1.0, True)
    got = T.distillation(student.to(DEV), ids.to(DEV), t.to(DEV), rest=True, reduction="none")
    close(got, c.loss, c.loss_err)
    _, dz = T.distillation_step(student.to(DEV), ids.to(DEV), t.to(DEV), rest=True,
                                reduction="sum")
    close(dz, *c.grad_bound(1.0, F32))


def test_the_rest_of_a_student_without_doubt(T):
    """Off the list the student has less than the smallest fp32: the gradient there still has the
    rest's own shape, where p / (sum of p) is 0 / 0."""
    v = 1000
    z = normal(2, v)
    ids = torch.tensor([[3, 500], [0, 999]])
    z.scatter_add_(1, ids, torch.full((2, 2), 300.0))
    t = torch.log(torch.tensor([[0.5, 0.3], [0.6, 0.1]]))
    c = L.Distill(z, ids, t, 1.0, True)
    assert float(c.dz[0, 10]) < 0 and float(c.loss[0]) > 50
    close(T.distillation(z.to(DEV), ids.to(DEV), t.to(DEV), rest=True, reduction="none"), c.loss,
          c.loss_err)
    dz = T.distillation_step(z.to(DEV), ids.to(DEV), t.to(DEV), rest=True, reduction="sum")[1]
    close(dz, *c.grad_bound(1.0, F32))


def test_no_teacher(T):
    z, ids, t = kd_case(5, 300, 4, BF16)
    ids[:] = 7
    ids[:, 1] = 3
    kw = dict(ignore_index=7)
    loss, dz = T.distillation_step(z.to(DEV), ids.to(DEV), t.to(DEV), **kw)
    assert torch.isnan(loss) and not dz.any()
    loss, dz = T.distillation_step(z.to(DEV), ids.to(DEV), t.to(DEV), reduction="sum", **kw)
    assert loss == 0 and not dz.any()
    assert T.distillation(z.to(DEV)[0], ids.to(DEV)[0], t.to(DEV)[0], **kw,
                          reduction="none").shape == ()


def test_distillation_gradient_against_differences(T):
    z, ids, t = kd_case(40, 3001, 12)
    d = torch.sign(normal(40, 3001, seed=9))
    kw = dict(temperature=1.5, rest=True, reduction="none")
    leaf = z.to(DEV).requires_grad_()
    ig, tg = ids.to(DEV), t.to(DEV)
    loss = T.distillation(leaf, ig, tg, **kw)
    (dz,) = torch.autograd.grad(loss.sum(), leaf)
    h = 2.0 ** -6
    with torch.no_grad():
        up = T.distillation(leaf + h * d.to(DEV), ig, tg, **kw).double()
        down = T.distillation(leaf - h * d.to(DEV), ig, tg, **kw).double()
    slope = (dz.double() * d.to(DEV)).sum(1)
    # third derivatives of lse and of the rest's along d: at most 2 / tau^3 each, times tau^2; each
    # loss is off by its bound, and z +- h d by half a last place of 16
    c = L.Distill(z, ids, t, 1.5, True)
    bound = h * h / 6 * 4 / 1.5 + (c.loss_err + 64 * E32) / h + (c.dz_err + 4 * E32 * c.dz.abs()
                                                                 ).sum(1)
    close((up - down) / (2 * h), slope.cpu(), bound)


def test_distillation_past_32_bit_offsets(T):
    n, v = 43000, 50257
    z = torch.zeros((n, v), dtype=BF16, device=DEV)
    ids = torch.tensor([9, 50256], device=DEV).repeat(n, 1)
    t = torch.log(torch.tensor([0.6, 0.3], device=DEV)).repeat(n, 1)
    z[-1, 9] = 12.0
    want = torch.zeros(1, v, dtype=BF16)
    want[0, 9] = 12.0
    c = L.Distill(want, ids[:1].cpu(), t[:1].cpu(), 1.0, True)
    loss = T.distillation(z, ids, t, rest=True, reduction="none")
    close(loss[-1:], c.loss, c.loss_err)
    _, dz = T.distillation_step(z, ids, t, rest=True, reduction="sum", inplace=True)
    close(dz[-1:], *c.grad_bound(1.0, BF16))


def test_distillation_refusals(T, Err):
    z, ids = torch.ones(4, 9, device=DEV), torch.zeros(4, 2, dtype=torch.int64, device=DEV)
    t = torch.zeros(4, 2, device=DEV)
    for call in (lambda: T.distillation(z.double(), ids, t),
                 lambda: T.distillation(z, ids.float(), t), lambda: T.distillation(z, ids.cpu(), t),
                 lambda: T.distillation(z, ids, t.cpu()), lambda: T.distillation(z, ids, t.double()),
                 lambda: T.distillation(z, ids[:3], t[:3]), lambda: T.distillation(z, ids, t[:, :1]),
                 lambda: T.distillation(z, ids[:, :0], t[:, :0]),
                 lambda: T.distillation(z, ids, t.requires_grad_()),
                 lambda: T.distillation(z, ids, t.detach(), temperature=-1.0),
                 lambda: T.distillation_step(z, ids, t.detach(), reduction="none"),
                 lambda: T.distillation_step(z.T, ids.repeat(3, 1)[:9], t.detach().repeat(3, 1)[:9],
                                             inplace=True),
                 lambda: T.distillation_step(z[:1].expand(4, 9), ids, t.detach(), inplace=True)):
        with pytest.raises(Err):
            call()


# ---- together ---------------------------------------------------------------------------------
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_student_learns_its_teachers_top_classes(T, rest, dtype):
    """The teacher's pass and the student's, with padding that the teacher's lists carry on."""
    tau, n, v, k = 2.0, 30, 5003, 24
    teacher, student = normal(n, v, dtype=dtype, std=3.0), normal(n, v, dtype=dtype, seed=1)
    y = torch.randint(0, v, (n,), generator=torch.Generator().manual_seed(2))
    y[-4:] = -100
    out = T.token_log_probs(teacher.to(DEV), y.to(DEV), top=k, temperature=tau)
    leaf = student.to(DEV).requires_grad_()
    loss = T.distillation(leaf, out.top_ids, out.top_log_probs, temperature=tau, rest=rest)
    (dz,) = torch.autograd.grad(loss, leaf)
    ids = L.top(teacher, k)
    ids[-4:] = -100
    t = out.top_log_probs.cpu()
    c = L.Distill(student, ids, t, tau, rest)
    want, err, count = c.mean()
    assert count == n - 4
    close(loss, want, err)
    close(dz, *c.grad_bound(1.0 / count, dtype))
    # the same logits: no divergence but for the teacher's roundings, which the bounds count
    same = T.distillation(teacher.to(DEV), out.top_ids, out.top_log_probs, temperature=tau,
                          rest=True, reduction="none")
    c = L.Distill(teacher, ids, t, tau, True)
    close(same, c.loss, c.loss_err)
    assert float(same.abs().max()) < 1e-4


def test_learning_from_rewards(T):
    """Log probabilities of a model's own tokens weighted with advantages, and an entropy bonus."""
    h, w = normal(64, 96, seed=1).to(DEV).requires_grad_(), normal(96, 2003, seed=2).to(DEV)
    y = torch.randint(0, 2003, (64,), generator=torch.Generator().manual_seed(0)).to(DEV)
    adv = normal(64, seed=3).to(DEV)
    out = T.token_log_probs(h @ w, y)
    loss = -(out.log_probs * adv).mean() - 0.01 * out.entropy.mean()
    (got,) = torch.autograd.grad(loss, h)
    hd = h.detach().cpu().double().requires_grad_()
    lp = torch.log_softmax(hd @ w.cpu().double(), 1)
    ent = -(lp.exp() * lp).sum(1)
    want = -(lp.gather(1, y.cpu()[:, None])[:, 0] * adv.cpu()).mean() - 0.01 * ent.mean()
    (dh,) = torch.autograd.grad(want, hd)
    # products of 96 and 2003 terms, logits up to 60 whose rounding is in every probability
    assert float((got.cpu().double() - dh).norm()) <= 2200 * 8 * E32 * float(dh.norm())


def test_on_another_stream(T):
    z, y = lp_case(64, 9009, BF16)
    _, ids, t = kd_case(64, 9009, 20)
    zg, yg, ig, tg = z.to(DEV), y.to(DEV), ids.to(DEV), t.to(DEV)

    def all_of():
        return (*T.token_log_probs(zg, yg, top=20), *T.distillation_step(zg, ig, tg, rest=True),
                T.distillation(zg, ig, tg))
    side = torch.cuda.Stream()
    here = all_of()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = all_of()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(here, there):
        assert torch.equal(a, b)


def test_in_a_captured_graph(T):
    """Every replay equals the eager calls on what the inputs hold then, gradients too; the
    graph's leaf is its own."""
    z, y = lp_case(100, 9001, BF16)
    _, ids, t = kd_case(100, 9001, 16)
    z, y, ids, t = z.to(DEV), y.to(DEV), ids.to(DEV), t.to(DEV)
    gh = normal(100).to(DEV)

    def step():
        leaf = z.detach().requires_grad_()
        out = T.token_log_probs(leaf, y, top=16)
        (dz,) = torch.autograd.grad([out.log_probs, out.entropy], leaf, [gh, gh])
        loss = T.distillation(leaf, out.top_ids, out.top_log_probs.detach(), temperature=1.2)
        (dk,) = torch.autograd.grad(loss, leaf)
        return (*(o.detach() for o in out), dz, loss.detach(), dk,
                *T.distillation_step(z, ids, t, rest=True))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for k in range(4):
        zz, yy = lp_case(100, 9001, BF16, seed=k)
        _, ii, tt = kd_case(100, 9001, 16, seed=k)
        z.copy_(zz), y.copy_(yy), ids.copy_(ii), t.copy_(tt)
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b), k


@pytest.mark.filterwarnings("ignore")
def test_compiled_programs_run_the_calls(T):
    z, y = lp_case(9, 300, F32)
    _, ids, t = kd_case(9, 300, 5)
    zg, yg, ig, tg = z.to(DEV).requires_grad_(), y.to(DEV), ids.to(DEV), t.to(DEV)

    def step(x):
        out = T.token_log_probs(x * 2, yg, top=3)
        return (out.log_probs.sum() + out.entropy.sum() + out.top_log_probs.sum()
                + T.distillation(x * 3, ig, tg))
    compiled = torch.compile(step, backend="aot_eager")
    a, b = step(zg), compiled(zg)
    assert torch.equal(a, b)
    assert torch.equal(*(torch.autograd.grad(x, zg)[0] for x in (a, b)))
    torch._dynamo.reset()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_values_below_the_normal_ones_keep_their_order(T, dtype):
    """Subnormal logits, and -0 among 0."""
    g = torch.Generator().manual_seed(0)
    z = torch.zeros(3, 4000)
    z[0] = (torch.randn(4000, generator=g) * 1e-39)
    z[1, ::2] = -0.0
    z[2] = -(torch.randint(0, 4, (4000,), generator=g) * 2.0 ** -133)
    z = z.to(dtype)
    for k in (3, 100):
        got = T.token_log_probs(z.to(DEV), top=k)
        assert torch.equal(got.top_ids.cpu(), L.top(z, k))


def test_an_ignored_token_that_is_a_class(T):
    """The lists of its rows are marked by what is no class, and others may name it."""
    z, _ = lp_case(6, 50, F32)
    z[:, 0] += 9.0
    y = torch.tensor([0, 3, 4, 0, 9, 1])
    out = T.token_log_probs(z.to(DEV), y.to(DEV), top=3, ignore_index=0)
    assert (out.top_ids == -100).all(1).tolist() == [True, False, False, True, False, False]
    assert out.top_ids[1, 0] == 0 and not out.entropy[[0, 3]].any()
    loss = T.distillation(z.to(DEV), out.top_ids, out.top_log_probs, rest=True, reduction="none")
    assert torch.isfinite(loss).all() and loss[0] == loss[3] == 0


def test_an_unknown_token_leaves_the_other_gradients(T):
    z, _ = lp_case(4, 300, F32)
    y = torch.tensor([5, 300, -1, 7])
    leaf = z.to(DEV).requires_grad_()
    out = T.token_log_probs(leaf, y.to(DEV), top=4)
    gh, gt = normal(4), normal(4, 4, seed=1)
    (dz,) = torch.autograd.grad([out.entropy, out.top_log_probs], leaf, [gh.to(DEV), gt.to(DEV)])
    close(dz, *L.log_probs_grad(z, y, out.top_ids.cpu(), None, gh, gt, 1.0, F32))


@pytest.mark.parametrize("rest", [False, True])
def test_ids_beyond_32_bits(T, rest):
    z, ids, t = kd_case(4, 300, 5, ragged=False)
    ids[0, 2], ids[2, 1], ids[3, 4] = 2 ** 32 + 7, -2 ** 40, 2 ** 31
    c = L.Distill(z, ids, t, 1.0, rest)
    got = T.distillation(z.to(DEV), ids.to(DEV), t.to(DEV), rest=rest, reduction="none")
    close(got, c.loss, c.loss_err)
    assert torch.isnan(got).tolist() == [True, False, True, True]


def test_as_many_classes_as_there_may_be(T, Err):
    """2^27 classes: all zero but a few, of which the last is one."""
    v = 1 << 27
    z = torch.zeros(1, v, dtype=F16, device=DEV)
    at = torch.tensor([v - 1, 12345, v // 2 + 3, v - 9])
    z[0, at.to(DEV)] = torch.tensor([9.0, 7.0, 8.0, 6.0], dtype=F16, device=DEV)
    total = float((v - 4) + torch.exp(torch.tensor([9.0, 8.0, 7.0, 6.0]).double()).sum())
    lse = torch.log(torch.tensor(total).double())
    y = torch.tensor([v - 1], device=DEV)
    out = T.token_log_probs(z, y, top=6)
    assert out.top_ids[0].tolist() == [v - 1, v // 2 + 3, 12345, v - 9, 0, 1]
    # a thread adds 2^17 terms in sequence
    bound = (v // 1024 + 100) * E32
    close(out.top_log_probs[0], torch.tensor([9.0, 8.0, 7.0, 6.0, 0.0, 0.0]).double() - lse, bound)
    close(out.log_probs, (9.0 - lse)[None], bound)
    t = torch.log(torch.tensor([[0.5, 0.25]], device=DEV))
    ids = at[None, :2].to(DEV)
    loss, dz = T.distillation_step(z, ids, t, rest=True, reduction="sum")
    p = torch.exp(torch.tensor([9.0, 7.0]).double() - lse)
    q = torch.tensor([0.5, 0.25]).double()
    rest = 1 - p.sum()
    want = (q * (q.log() - p.log())).sum() + 0.25 * (torch.log(torch.tensor(0.25).double())
                                                     - torch.log(rest))
    close(loss, want, 3 * bound + 20 * E32)
    got = dz[0, at[:2].to(DEV)].cpu().double()
    assert float((got - (p - q)).abs().max()) <= 2 * bound + 2.0 ** -11
    with pytest.raises(Err, match="bad arguments"):
        T.token_log_probs(torch.zeros(1, dtype=F16, device=DEV).expand(v + 1)[None])


def test_many_rows_of_few_classes(T):
    n, v = (1 << 19) + 3, 9
    z = normal(n, v, dtype=BF16, std=2.0)
    y = torch.arange(n) % v
    ids = torch.stack([y, (y + 4) % v], 1)
    t = torch.log(torch.tensor([0.5, 0.2])).repeat(n, 1)
    ids[5::7] = -100
    some = torch.cat([torch.arange(500), torch.arange(n - 500, n)])
    out = T.token_log_probs(z.to(DEV), y.to(DEV), top=2)
    ref, top = L.log_probs(z[some], y[some], 2)
    close(out.log_probs[some.to(DEV)], *ref["log_probs"])
    assert torch.equal(out.top_ids.cpu(), L.top(z, 2))
    c = L.Distill(z, ids, t, 1.0, True)
    loss, err, count = c.mean()
    got, dz = T.distillation_step(z.to(DEV), ids.to(DEV), t.to(DEV), rest=True)
    close(got, loss, err)
    close(dz, *c.grad_bound(1.0 / count, BF16))


@pytest.mark.parametrize("n", [255, 256, 257, 700])
def test_rows_with_a_teacher_are_counted(T, n):
    """By the rows' own launch, or by one before it."""
    z, ids, t = kd_case(n, 130, 3, ragged=False)
    ids[::3, 0] = -100
    c = L.Distill(z, ids, t, 1.0, False)
    loss, err, count = c.mean()
    got, dz = T.distillation_step(z.to(DEV), ids.int().to(DEV), t.to(DEV))
    close(got, loss, err)
    close(dz, *c.grad_bound(1.0 / count, F32))
    close(T.distillation(z.to(DEV), ids.to(DEV), t.to(DEV)), loss, err)


def test_logits_past_the_caches(T):
    """The loads and stores of logits of 400 MB, a few rows of which are compared."""
    n, v = 4300, 50257
    z = torch.randn(n, v, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).to(BF16)
    _, ids, t = kd_case(n, v, 6, ragged=False)
    y = ids[:, 3].clamp(min=0)
    some = torch.tensor([0, 1, 2, 777, n - 2, n - 1])
    zs = z[some.to(DEV)].cpu()
    c = L.Distill(zs, ids[some], t[some], 1.0, True)
    ig, tg = ids.to(DEV), t.to(DEV)
    leaf = z.clone().requires_grad_()
    (g,) = torch.autograd.grad(T.distillation(leaf, ig, tg, rest=True, reduction="sum"), leaf)
    close(g[some.to(DEV)], *c.grad_bound(1.0, BF16))
    out = T.token_log_probs(leaf, y.to(DEV), top=10)
    ref, top = L.log_probs(zs, y[some], 10)
    close(out.entropy[some.to(DEV)], *ref["entropy"])
    assert torch.equal(out.top_ids[some.to(DEV)].cpu(), top)
    gy = normal(n)
    (g,) = torch.autograd.grad(out.log_probs, leaf, gy.to(DEV))
    close(g[some.to(DEV)], *L.log_probs_grad(zs, y[some], None, gy[some], None, None, 1.0, BF16))
    close(T.distillation(z, ig, tg, rest=True, reduction="none")[some.to(DEV)], c.loss, c.loss_err)
    _, dz = T.distillation_step(z, ig, tg, rest=True, reduction="sum", inplace=True)
    close(dz[some.to(DEV)], *c.grad_bound(1.0, BF16))


def test_a_models_step_on_a_teacher(T):
    """The benchmark's GPT-2 as a student of another one, in place, against torch's operators in
    fp32.  As there, each gradient differs by the rounding of sums of some thousand fp32 terms
    (2^-24 each, relative to its norm) at each of a dozen products on its way."""
    import bench
    tok = torch.randint(0, 517, (3, 41), generator=torch.Generator().manual_seed(0)).to(DEV)
    x, y = tok[:, :-1], tok[:, 1:].clone()
    y[2, 30:] = -100                        # padding
    torch.manual_seed(1)
    teacher = bench._gpt2(517, 64, 64, 2, 4).to(DEV)
    with torch.no_grad():
        zt = teacher.logits(x) * 3.0        # (of a random model, all classes are nearly alike)
        top = T.token_log_probs(zt, y, top=16, temperature=2.0)
    got = {}
    for ops in ("torch", "hip"):
        torch.manual_seed(0)
        m = bench._gpt2(517, 64, 64, 2, 4, ops).to(DEV)
        z = m.logits(x)
        if ops == "hip":
            loss, dz = T.distillation_step(z, top.top_ids, top.top_log_probs, temperature=2.0,
                                           rest=True, inplace=True)
            z.backward(dz)
        else:
            live = y != -100
            lp = torch.log_softmax(zt / 2, -1)
            at = torch.topk(lp, 16, -1)[1]
            log_q, log_p = lp.gather(-1, at), torch.log_softmax(z / 2, -1)
            q = log_q.exp()
            inside = torch.zeros_like(lp, dtype=torch.bool).scatter_(-1, at, True)
            left = lp.exp().masked_fill(inside, 0).sum(-1)
            log_r = torch.logsumexp(log_p.masked_fill(inside, -torch.inf), -1)
            kl = (q * (log_q - log_p.gather(-1, at))).sum(-1) + left * (left.log() - log_r)
            loss = 4 * kl[live].mean()
            loss.backward()
        got[ops] = float(loss.detach()), {n: p.grad for n, p in m.named_parameters()}
    (a, ga), (b, gb) = got["torch"], got["hip"]
    assert abs(a - b) <= 1e-4 * a
    assert ga.keys() == gb.keys()
    for n in ga:
        assert float((ga[n] - gb[n]).norm()) <= 12 * 2000 * E32 * float(ga[n].norm()), n


@pytest.mark.parametrize("v", [1500, 9003, 50257, 66001, 131077])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_top_classes_among_equal_ones(T, v, dtype):
    """Equal classes at the end, in the second half, behind a few larger ones, in lumps; masks that
    leave fewer than are asked for."""
    g = torch.Generator().manual_seed(v)
    inf = float("inf")
    z = torch.randn(12, v, generator=g).clamp(max=3.0)
    z[0] = -1.0
    z[0, -1100:] = 5.0
    z[1, v // 2:] = 5.0
    z[2, v // 2 + 7:] = torch.where(torch.rand(v - v // 2 - 7, generator=g) < 0.5, 5.0, -1.0)
    z[3, v // 3:] = 4.0
    z[3, torch.randperm(v, generator=g)[:60]] = torch.arange(60.0) + 5.0
    z[4, :700] = 6.0 + torch.rand(min(v, 700), generator=g)
    z[5, 20:] = -inf
    z[6] = -inf
    z[6, torch.randperm(v, generator=g)[:100]] = 2.0
    z[7, :] = torch.arange(v).remainder(v // 7 + 1).float() / 64
    z[8] = torch.arange(v).div(900, rounding_mode="floor").float()
    z[9] = -torch.arange(v).div(900, rounding_mode="floor").float()
    z[10, ::2] = -inf
    z[11] = -torch.finfo(dtype).max
    z[11, 3] = torch.finfo(dtype).max
    z = z.to(dtype)
    for k in (1, 20, 64, 65, 101, 256):
        got = T.token_log_probs(z.to(DEV), top=k)
        assert torch.equal(got.top_ids.cpu(), L.top(z, k)), k
        check_log_probs(got, z, None, k, 1.0, k)
    many = z.repeat(60, 1).to(DEV)          # more rows than fit at a time
    got = T.token_log_probs(many, top=64)
    assert torch.equal(got.top_ids.cpu(), L.top(z, 64).repeat(60, 1))


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("v,k", [(60, 20), (600, 3), (9001, 70), (50257, 64), (140001, 300)])
def test_entries_left_out_by_a_class(T, v, k, rest):
    """An ignore_index that is a class: its entries are left out wherever they stand, and so is
    -100, by which token_log_probs then marks its lists."""
    none = 11
    z, ids, t = kd_case(12, v, k, cover=0.8, ragged=False)
    z[:, none] += 6.0                       # a class that counts
    ids = torch.where(ids == none, none + 1, ids)
    ids[0, k // 2] = none                   # in the middle
    ids[2, -1] = none                       # at the end
    ids[3, 1:] = none                       # all but the first
    ids[4, 0] = none                        # no teacher
    ids[5, -1] = -100
    ids[7, 1] = none
    ids[7, -1] = -100
    ids[8] = none
    same = torch.where(ids == -100, none, ids)
    c = L.Distill(z, same, t, 1.5, rest, none)
    assert c.live.tolist() == [r not in (1, 4, 6, 8, 11) for r in range(12)]
    assert torch.isfinite(c.loss).all()
    loss, err, count = c.mean()
    kw = dict(temperature=1.5, rest=rest, ignore_index=none)
    zg, tg = z.to(DEV), t.to(DEV)
    for ig in (ids.to(DEV), ids.int().to(DEV)):
        close(T.distillation(zg, ig, tg, reduction="none", **kw), c.loss, c.loss_err)
        close(T.distillation(zg, ig, tg, **kw), loss, err)
        got, dz = T.distillation_step(zg, ig, tg, **kw)
        close(got, loss, err)
        close(dz, *c.grad_bound(1.0 / count, F32))
        work = zg.clone()
        got, dz = T.distillation_step(work, ig, tg, reduction="sum", inplace=True, **kw)
        close(got, loss * count, err * count)
        close(dz, *c.grad_bound(1.0, F32))
        leaf = zg.clone().requires_grad_()
        (dz,) = torch.autograd.grad(T.distillation(leaf, ig, tg, **kw), leaf)
        close(dz, *c.grad_bound(1.0 / count, F32))


@pytest.mark.parametrize("rest", [False, True])
def test_a_teachers_padding_that_is_a_class(T, rest):
    """The same ignore_index, a class, in the teacher's pass and in the student's."""
    z, y = normal(300, 500, std=2.0), torch.arange(300) % 40
    z[3::4, 0] += 9.0                       # class 0 at the head of some lists
    student = normal(300, 500, seed=1)
    out = T.token_log_probs(z.to(DEV), y.to(DEV), top=8, ignore_index=0)
    ids = L.top(z, 8)
    ids[y == 0] = 0
    c = L.Distill(student, ids, out.top_log_probs.cpu(), 1.0, rest, 0)
    loss, err, count = c.mean()
    assert count == int(((y != 0) & (ids[:, 0] != 0)).sum()) and torch.isfinite(loss)
    kw = dict(rest=rest, ignore_index=0)
    got, dz = T.distillation_step(student.to(DEV), out.top_ids, out.top_log_probs, **kw)
    close(got, loss, err)
    close(dz, *c.grad_bound(1.0 / count, F32))
    leaf = student.to(DEV).requires_grad_()
    got = T.distillation(leaf, out.top_ids, out.top_log_probs, **kw)
    close(got, loss, err)
    close(torch.autograd.grad(got, leaf)[0], *c.grad_bound(1.0 / count, F32))


@pytest.mark.parametrize("n,v,k", [(700, 300, 64), (700, 70, 64), (40, 9001, 33), (12, 140001, 64)])
def test_lists_that_one_wave_marks(T, n, v, k):
    """Up to 64 entries: one wave's lanes clear the marks of a row, and others of them set these;
    classes in a lump, so that lanes share words, some of them twice."""
    z, ids, t = kd_case(n, v, k, cover=0.7, ragged=False)
    near = (torch.arange(k) + torch.arange(n)[:, None]) % min(v, 97)
    near[::3, 1] = near[::3, 0]
    near[::7, -1] = near[::7, k // 2]
    ids = torch.where(ids >= 0, near, ids)
    c = L.Distill(z, ids, t, 1.0, True)
    zg, ig, tg = z.to(DEV), ids.to(DEV), t.to(DEV)
    for _ in range(3):
        close(T.distillation(zg, ig, tg, rest=True, reduction="none"), c.loss, c.loss_err)
        close(T.distillation_step(zg, ig, tg, rest=True, reduction="sum")[1],
              *c.grad_bound(1.0, F32))


@pytest.mark.parametrize("n,v,dtype", [(4300, 50257, BF16), (3100, 33001, F32), (26000, 8009, BF16)])
def test_log_probs_past_the_caches(T, n, v, dtype):
    """Logits of more than 384 MiB without a gradient: rows held by a workgroup of either size, and
    streamed ones; those whose top is searched for among them."""
    assert n * v * dtype.itemsize >= 384 << 20
    z = torch.randn(n, v, device=DEV, generator=torch.Generator(device=DEV).manual_seed(2))
    z = z.mul_(2.0).to(dtype)
    z[1] = 0.0
    z[2, 20:] = -float("inf")
    z[3, v // 2:] = 9.0
    y = torch.randint(0, v, (n,), generator=torch.Generator().manual_seed(3))
    y[4] = -100
    some = torch.tensor([0, 1, 2, 3, 4, 5, n // 2, n - 2, n - 1])
    y[2] = 7
    zs, ys = z[some.to(DEV)].cpu(), y[some]
    for k in (0, 1, 30, 200):
        want, ids = L.log_probs(zs, ys, k)
        got = T.token_log_probs(z, y.to(DEV), top=k)
        for name, (value, bound) in want.items():
            close(getattr(got, name)[some.to(DEV)], value, bound.nan_to_num(0.0, 0.0, 0.0),
                  (k, name))
        if k:
            assert torch.equal(got.top_ids[some.to(DEV)].cpu(), ids), k


def test_as_many_rows_as_there_may_be(T, Err):
    n, v, k = (1 << 22) - 1, 130, 129
    z = torch.randn(n, v, device=DEV, generator=torch.Generator(device=DEV).manual_seed(2)).to(BF16)
    some = torch.cat([torch.arange(50), torch.arange(n - 50, n)])
    at = some.to(DEV)
    zs = z[at].cpu()
    y = torch.arange(n, device=DEV) % v
    want, ids = L.log_probs(zs, y[at].cpu(), k)
    out = T.token_log_probs(z, y, top=k)
    for name, (value, bound) in want.items():
        close(getattr(out, name)[at], value, bound, name)
    assert torch.equal(out.top_ids[at].cpu(), ids)
    leaf = z.requires_grad_()
    gh = normal(100)
    full = torch.zeros(n, device=DEV)
    full[at] = gh.to(DEV)
    del out
    (dz,) = torch.autograd.grad(T.token_log_probs(leaf, y).entropy, leaf, full)
    close(dz[at], *L.log_probs_grad(zs, None, None, None, gh, None, 1.0, BF16))
    z = z.detach()
    ids = torch.stack([y, (y + 4) % v], 1)
    ids[5::7, 0] = -100
    t = torch.log(torch.tensor([0.5, 0.2], device=DEV)).repeat(n, 1)
    c = L.Distill(zs, ids[at].cpu(), t[at].cpu(), 1.0, True)
    close(T.distillation(z, ids, t, rest=True, reduction="none")[at], c.loss, c.loss_err)
    count = n - len(range(5, n, 7))
    (dz,) = torch.autograd.grad(T.distillation(leaf, ids, t, rest=True), leaf)
    close(dz[at], *c.grad_bound(1.0 / count, BF16))
    dz = T.distillation_step(z, ids, t, rest=True, grad_scale=1e6, inplace=True)[1]
    close(dz[at], *c.grad_bound(1e6 / count, BF16))
    more = z[:1].expand(n + 1, v)
    for call in (lambda: T.token_log_probs(more),
                 lambda: T.distillation(more, ids[:1].expand(n + 1, 2), t[:1].expand(n + 1, 2))):
        with pytest.raises(Err, match="bad arguments"):
            call()


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("n,v,dtype", [(26000, 8009, BF16), (1700, 131077, BF16), (1600, 70001, F32),
                                       (900, 120001, F32)])
def test_distillation_past_the_caches(T, n, v, dtype, rest):
    """Logits of more than 384 MiB: rows held by workgroups of each size, and streamed ones."""
    assert n * v * dtype.itemsize >= 384 << 20
    k = 40
    z = torch.randn(n, v, device=DEV, generator=torch.Generator(device=DEV).manual_seed(2))
    z = z.mul_(2.0).to(dtype)
    ids = (torch.arange(n)[:, None] * 37 + torch.arange(k) * (v // 41)) % v
    ids[1::5] = -100
    ids[0, 3] = ids[0, 2]
    ids[2, 7:] = -100
    t = torch.log_softmax(normal(n, k, std=2.0, seed=4), 1) - 0.1
    some = torch.tensor([0, 1, 2, 3, 4, 7, n // 2, n - 3, n - 2, n - 1])
    at = some.to(DEV)
    c = L.Distill(z[at].cpu(), ids[some], t[some], 1.4, rest)
    count = int((ids[:, 0] >= 0).sum())
    ig, tg, kw = ids.to(DEV), t.to(DEV), dict(temperature=1.4, rest=rest)
    close(T.distillation(z, ig, tg, reduction="none", **kw)[at], c.loss, c.loss_err)
    dz = T.distillation_step(z, ig, tg, **kw)[1]
    close(dz[at], *c.grad_bound(1.0 / count, dtype))
    leaf = z.clone().requires_grad_()
    (dz,) = torch.autograd.grad(T.distillation(leaf, ig, tg, **kw), leaf)
    close(dz[at], *c.grad_bound(1.0 / count, dtype))
    dz = T.distillation_step(z, ig, tg, reduction="sum", inplace=True, **kw)[1]
    close(dz[at], *c.grad_bound(1.0, dtype))


def test_two_graphs_of_one_memory_pool(T):
    """Rows counted by a launch of their own, in place and through autograd, in two graphs that
    share their memory and are replayed in turn with eager work between."""
    n, v, k = 700, 4099, 12
    cases = []
    for seed in (0, 1):
        z, ids, t = kd_case(n, v, k, BF16, seed=seed)
        cases.append([x.to(DEV) for x in (z, ids, t)])

    def step(z, ids, t):
        top = T.token_log_probs(z, top=5)
        leaf = z.detach().requires_grad_()
        loss = T.distillation(leaf, ids, t, rest=True)
        (g,) = torch.autograd.grad(loss, leaf)
        work = z.clone()
        mean, dz = T.distillation_step(work, ids, t, inplace=True)
        return (*top[1:], loss.detach(), g, mean, dz)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*cases[0])
    torch.cuda.current_stream().wait_stream(side)
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    outs = []
    for graph in (first, second):
        with torch.cuda.graph(graph, pool=first.pool() if graph is second else None):
            outs.append(step(*cases[len(outs)]))
    for turn in range(4):
        for i, graph in enumerate((first, second)):
            z, ids, t = kd_case(n, v, k, BF16, seed=10 + 2 * turn + i)
            for a, b in zip(cases[i], (z, ids, t)):
                a.copy_(b)
            want = step(*cases[i])
            torch.cuda.synchronize()
            graph.replay()
            got = [x.clone() for x in outs[i]]
            torch.cuda.synchronize()
            for a, b in zip(got, want):
                assert torch.equal(a, b), (turn, i)


def test_calls_on_two_streams_at_once(T):
    """From two threads with a stream each."""
    import threading
    data, want, got = [], [], [None, None]
    for seed in (0, 1):
        z, ids, t = kd_case(900, 9003, 20, BF16, seed=seed)
        data.append([x.to(DEV) for x in (z, ids, t)])

    def calls(z, ids, t):
        out = []
        for _ in range(10):
            out = [*T.token_log_probs(z, ids[:, 2].clamp(min=0), top=20),
                   *T.distillation_step(z, ids, t, rest=True)]
            leaf = z.detach().requires_grad_()
            out.append(torch.autograd.grad(T.distillation(leaf, ids, t), leaf)[0])
        return out
    for d in data:
        want.append(calls(*d))
    torch.cuda.synchronize()

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            got[i] = calls(*data[i])
            torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=run, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for g, w in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(g, w))


def test_a_repeated_forward_pass(T):
    """Activation checkpointing runs the calls again in the backward pass."""
    from torch.utils.checkpoint import checkpoint
    h, w = normal(30, 16, seed=1).to(DEV).requires_grad_(), normal(16, 600, seed=2).to(DEV)
    _, ids, t = kd_case(30, 600, 8)
    y, ids, t = ids[:, 1].clamp(min=0).to(DEV), ids.to(DEV), t.to(DEV)

    def f(h):
        out = T.token_log_probs(h @ w, y, top=4)
        return (out.log_probs.sum() + out.entropy.sum() + out.top_log_probs.sum()
                + T.distillation(h @ w, ids, t, rest=True))
    want = torch.autograd.grad(f(h), h)[0]
    assert torch.equal(torch.autograd.grad(checkpoint(f, h, use_reentrant=False), h)[0], want)
