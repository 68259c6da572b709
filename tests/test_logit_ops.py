"""CPU checks of the log probabilities and of distillation: the plain forms against autograd and
differences, the host's checks of arguments (no kernel is launched), and what autograd and traces
see."""

import ctypes

import pytest
import torch

import logit_ref as L
from train_ref import E32

F64 = torch.float64


def _case(n=5, v=40, k=6, seed=0):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(n, v, generator=g, dtype=F64) * 2
    ids = torch.stack([torch.randperm(v, generator=g)[:k] for _ in range(n)])
    t = torch.log_softmax(torch.randn(n, k, generator=g, dtype=F64), -1) - 0.3
    return z, torch.randint(0, v, (n,), generator=g), ids, t


@pytest.mark.parametrize("tau", [1.0, 0.6, 3.0])
def test_reference_log_probs_follow_their_definition(tau):
    z, y, _, _ = _case()
    x = (z / tau).requires_grad_()
    lp = torch.log_softmax(x, 1)
    h = torch.distributions.Categorical(logits=x).entropy()
    out, ids = L.log_probs(z, y, 4, tau)
    assert torch.allclose(out["log_probs"][0], lp.gather(1, y[:, None])[:, 0], atol=1e-12)
    assert torch.allclose(out["entropy"][0], h, atol=1e-12)
    top = torch.topk(lp, 4, 1)
    assert torch.equal(ids, top[1]) and torch.allclose(out["top_log_probs"][0], top[0])
    g = torch.Generator().manual_seed(1)
    gy, gh = torch.randn(5, generator=g, dtype=F64), torch.randn(5, generator=g, dtype=F64)
    gt = torch.randn(5, 4, generator=g, dtype=F64)
    total = (lp.gather(1, y[:, None])[:, 0] * gy).sum() + (h * gh).sum() \
        + (lp.gather(1, ids) * gt).sum()
    want = torch.autograd.grad(total, x)[0] / tau
    got, bound = L.log_probs_grad(z, y, ids, gy, gh, gt, tau, torch.float32)
    assert torch.allclose(got, want, atol=1e-12) and bool((bound < 1e-3).all())


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("tau", [1.0, 2.5])
def test_reference_distillation_follows_its_definition(rest, tau):
    z, _, ids, t = _case()
    ids[1, 3], ids[2, 1] = -100, ids[2, 0]   # one left out, one listed twice
    c = L.Distill(z, ids, t, tau, rest)
    z = z.requires_grad_()
    p = torch.softmax(z / tau, 1)
    loss = 0
    for row in range(5):
        some = ids[row] != -100
        i, w = ids[row][some], t[row][some]
        q = torch.exp(w) if rest else torch.softmax(w, 0)
        part = (q * (q.log() - p[row, i].log())).sum()
        if rest:
            left, r = 1 - q.sum(), 1 - p[row, i.unique()].sum()
            part = part + left * (left.log() - r.log())
        loss = loss + part * tau ** 2
        assert abs(float(part) * tau ** 2 - float(c.loss[row])) < 1e-10
    assert torch.allclose(torch.autograd.grad(loss, z)[0], c.dz, atol=1e-10)
    assert bool((c.dz_err < 1e-3).all()) and bool((c.loss_err < 1e-3).all())


@pytest.mark.parametrize("rest", [False, True])
def test_reference_distillation_against_differences(rest):
    z, _, ids, t = _case()
    d = torch.sign(torch.randn(z.shape, generator=torch.Generator().manual_seed(4), dtype=F64))
    h = 1e-5
    c, up, down = (L.Distill(z + e * d, ids, t, 1.5, rest) for e in (0, h, -h))
    assert torch.allclose((up.loss - down.loss) / (2 * h), (c.dz * d).sum(1), atol=1e-7)


def test_a_teacher_of_its_own_has_no_divergence():
    z = _case()[0]
    ids = L.top(z, 7)
    t = torch.log_softmax(z / 2, 1).gather(1, ids)
    c = L.Distill(z, ids, t, 2.0, True)
    assert float(c.loss.abs().max()) < 1e-12 and float(c.dz.abs().max()) < 1e-12


@pytest.fixture(scope="module")
def lib():
    from defmuon_amd import _native
    return _native.load()


def test_entry_points_refuse_without_launching(lib):
    one = ctypes.c_void_p(256)   # never read: every call below is refused on the host

    def lp(**kw):
        a = dict(z=one, dt=0, rows=2, v=9, zs=9, y=one, tau=1.0, top=3, lp=one, h=one, tl=one,
                 ti=one)
        a.update(kw)
        return lib.dmh_log_probs(None, a["z"], a["dt"], a["rows"], a["v"], a["zs"], a["y"], 1,
                                 -100, a["tau"], a["top"], a["lp"], a["h"], a["tl"], a["ti"], None)
    nan = float("nan")
    for bad in (dict(z=None), dict(dt=3), dict(rows=-1), dict(rows=1 << 22), dict(v=0),
                dict(v=(1 << 27) + 1), dict(zs=-1), dict(tau=0.0), dict(tau=-1.0), dict(tau=nan),
                dict(tau=1e7), dict(top=-1), dict(top=10), dict(v=400, top=257), dict(lp=None),
                dict(tl=None), dict(ti=None)):
        assert lp(**bad) == 1, bad
        assert b"dmh_log_probs" in lib.dmh_last_error()
    assert lp(rows=0, z=None) == 0

    def lg(**kw):
        a = dict(z=one, dt=0, rows=2, v=9, zs=9, y=one, tau=1.0, top=3, ti=one, st=one, gy=one,
                 gt=one, dz=one, ds=9)
        a.update(kw)
        return lib.dmh_log_probs_grad(None, a["z"], a["dt"], a["rows"], a["v"], a["zs"], a["y"], 1,
                                      -100, a["tau"], a["top"], a["ti"], a["st"], a["gy"], None,
                                      a["gt"], a["dz"], a["ds"])
    for bad in (dict(z=None), dict(dt=3), dict(rows=1 << 22), dict(v=0), dict(zs=-1), dict(ds=-1),
                dict(tau=nan), dict(top=10), dict(y=None), dict(ti=None), dict(st=None),
                dict(dz=None)):
        assert lg(**bad) == 1, bad
        assert b"dmh_log_probs_grad" in lib.dmh_last_error()
    assert lg(rows=0) == 0

    def kd(**kw):
        a = dict(z=one, dt=0, rows=2, v=9, zs=9, ids=one, k=3, t=one, tt=0, tau=1.0, red=1,
                 loss=one, count=one, ds=9, ws=one, nb=1 << 20)
        a.update(kw)
        return lib.dmh_distill(None, a["z"], a["dt"], a["rows"], a["v"], a["zs"], a["ids"], 1,
                               a["k"], a["t"], a["tt"], -100, a["tau"], 0, a["red"], 1.0,
                               a["loss"], a["count"], None, None, a["ds"], a["ws"], a["nb"])
    for bad in (dict(z=None), dict(ids=None), dict(t=None), dict(loss=None), dict(count=None),
                dict(dt=3), dict(tt=-1), dict(rows=-1), dict(rows=1 << 22), dict(v=0),
                dict(v=1 << 31), dict(zs=-1), dict(ds=-1), dict(k=0), dict(k=1025), dict(tau=0.0),
                dict(tau=nan), dict(red=3), dict(red=-1)):
        assert kd(**bad) == 1, bad
        assert b"dmh_distill" in lib.dmh_last_error()
    assert kd(ws=None) == 2 and kd(nb=1) == 2
    assert b"workspace" in lib.dmh_last_error()
    assert kd(rows=0, red=0) == 0

    def kg(**kw):
        a = dict(z=one, dt=0, rows=2, v=9, zs=9, ids=one, k=3, t=one, tt=0, tau=1.0, st=one,
                 go=one, dz=one, ds=9)
        a.update(kw)
        return lib.dmh_distill_grad(None, a["z"], a["dt"], a["rows"], a["v"], a["zs"], a["ids"], 1,
                                    a["k"], a["t"], a["tt"], -100, a["tau"], a["st"], None,
                                    a["go"], 0, a["dz"], a["ds"])
    for bad in (dict(z=None), dict(ids=None), dict(t=None), dict(st=None), dict(go=None),
                dict(dz=None), dict(dt=5), dict(tt=5), dict(rows=1 << 22), dict(v=0), dict(k=0),
                dict(k=1025), dict(zs=-2), dict(ds=-2), dict(tau=nan)):
        assert kg(**bad) == 1, bad
        assert b"dmh_distill_grad" in lib.dmh_last_error()
    assert kg(rows=0) == 0
    nb = ctypes.c_size_t()
    size = lib.dmh_distill_workspace_size
    assert size(-1, ctypes.byref(nb)) == 1 and size(1, None) == 1
    assert size(1000, ctypes.byref(nb)) == 0 and nb.value == 4 * (2 * 1000 + 64)


def test_no_cpu_fallback():
    from defmuon_amd import train_ops as T
    from defmuon_amd._native import NativeError
    z, ids, t = torch.randn(4, 8), torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 2)
    for call in (lambda: T.token_log_probs(z, ids[:, 0]), lambda: T.token_log_probs(z, top=2),
                 lambda: T.distillation(z, ids, t), lambda: T.distillation_step(z, ids, t)):
        with pytest.raises(NativeError, match="GPU"):
            call()


@pytest.fixture
def stand_in(monkeypatch):
    """train_ops on CPU tensors: plain forms in place of the launches, through their memory."""
    from defmuon_amd import _native, train_ops as T
    seen = {}

    def log_probs(z, rows, y, ignore, tau, top, lp, ent, top_lp, ids, stats):
        assert all(type(n) is int for n in rows)
        out, at = L.log_probs(z.detach().view(rows[:2]), None if y is None else y.view(-1), top,
                              tau, ignore)
        for name, t in (("log_probs", lp), ("entropy", ent), ("top_log_probs", top_lp)):
            if t is not None:
                t.detach().numpy()[...] = out[name][0].view(t.shape).float().numpy()
        if top:
            ids.numpy()[...] = at.view(ids.shape).numpy()

    def log_probs_grad(z, rows, y, ignore, tau, ids, stats, grads, dz, stride):
        seen["grads"] = grads
        gy, gh, gt = grads
        dz.numpy()[...] = L.log_probs_grad(z.detach(), y, ids, gy, gh, gt, tau, torch.float32,
                                           ignore)[0].float().numpy()

    def distill(z, rows, ids, t, ignore, tau, rest, red, scale, loss, dz, stride, keep):
        c = L.Distill(z.detach(), ids, t.detach(), tau, rest, ignore)
        n = int(c.live.sum()) if red == 1 else 1
        loss.detach().numpy()[...] = (c.loss if red == 0 else c.loss.sum() / n).float().numpy()
        if dz is not None:
            dz.numpy()[...] = (c.dz * scale / n).float().numpy()
        return torch.zeros(1)

    def distill_grad(z, rows, ids, t, ignore, tau, red, stats, g, dz, stride):
        c = L.Distill(z.detach(), ids, t.detach(), tau, False, ignore)
        n = int(c.live.sum()) if red == 1 else 1
        dz.numpy()[...] = (c.dz / n * g.reshape(-1, 1)).float().numpy()
    monkeypatch.setattr(T, "_float", lambda *a: None)
    for f in (log_probs, log_probs_grad, distill, distill_grad):
        monkeypatch.setattr(_native, f.__name__, f)
    return T, seen


def test_outputs_and_their_gradients(stand_in):
    T, seen = stand_in
    z, y, _, _ = _case()
    z = z.float().requires_grad_()
    out = T.token_log_probs(z, y, top=3, temperature=0.5)
    assert out._fields == ("log_probs", "entropy", "top_log_probs", "top_ids")
    assert [t.requires_grad for t in out] == [True, True, True, False]
    torch.autograd.grad(out.entropy.sum(), z)
    assert [g is None for g in seen["grads"]] == [True, False, True]
    out = T.token_log_probs(z, y, top=3)
    torch.autograd.grad(out.log_probs.sum() + out.top_log_probs.sum(), z)
    assert [g is None for g in seen["grads"]] == [False, True, False]
    out = T.token_log_probs(z.detach(), y)
    assert out.top_ids is out.top_log_probs is None and not out.entropy.requires_grad
    out = T.token_log_probs(z, top=2)
    assert out.log_probs is None
    ids = out.top_ids
    loss = out.top_log_probs.sum()
    ids += 1   # what the backward pass needs
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_refusals(stand_in):
    from defmuon_amd._native import NativeError
    T, _ = stand_in
    z, y, ids, t = _case()
    z, t = z.float(), t.float()
    wide = torch.zeros(2, 300)
    for call in (lambda: T.token_log_probs(z, y[:3]), lambda: T.token_log_probs(z, y.float()),
                 lambda: T.token_log_probs(z, top=41), lambda: T.token_log_probs(z, top=-1),
                 lambda: T.token_log_probs(wide, top=257), lambda: T.token_log_probs(z[0, 0]),
                 lambda: T.token_log_probs(z[:, :0]),
                 lambda: T.token_log_probs(z, temperature=0.0),
                 lambda: T.token_log_probs(z, temperature=float("nan")),
                 lambda: T.token_log_probs(z, temperature=-1.0),
                 lambda: T.distillation(z, ids[:3], t[:3]), lambda: T.distillation(z, ids[0], t[0]),
                 lambda: T.distillation(z, ids, t[:, :2]), lambda: T.distillation(z, ids.float(), t),
                 lambda: T.distillation(z, ids[:, :0], t[:, :0]),
                 lambda: T.distillation(z, ids.repeat(1, 171)[:, :1025], t.repeat(1, 171)[:, :1025]),
                 lambda: T.distillation(z, ids, t, temperature=1e9),
                 lambda: T.distillation(z, ids, t, reduction="max"),
                 lambda: T.distillation(z, ids, t.clone().requires_grad_()),
                 lambda: T.distillation_step(z, ids, t, reduction="none"),
                 lambda: T.distillation_step(z[:1].expand(5, 40), ids, t, inplace=True)):
        with pytest.raises(NativeError):
            call()
    with torch.no_grad():   # no gradient is lost
        T.distillation(z, ids, t.clone().requires_grad_())


def test_steps_in_place_are_seen_by_autograd(stand_in):
    T, _ = stand_in
    h, w = torch.randn(5, 8, requires_grad=True), torch.randn(8, 40)
    _, _, ids, t = _case()
    t = t.float()
    want = torch.autograd.grad(z := h @ w, h, T.distillation_step(z, ids, t)[1])[0]
    (g,) = torch.autograd.grad(T.distillation(h @ w, ids, t), h)
    assert torch.allclose(g, want, atol=1e-6)
    z = h @ w
    loss, dz = T.distillation_step(z, ids, t, inplace=True)
    assert dz.data_ptr() == z.data_ptr() and z._version == 1
    assert torch.equal(torch.autograd.grad(z, h, dz)[0], want)
    z = torch.tanh(h @ w)
    dz = T.distillation_step(z, ids, t, inplace=True)[1]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward(dz)


@pytest.mark.filterwarnings("ignore::DeprecationWarning")
def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fwd
    from defmuon_amd import train_ops as T
    from defmuon_amd._native import NativeError
    z, y, ids, t = _case()
    z, t = z.float(), t.float()
    with fwd.dual_level():
        def dual(x, grad=False):
            return fwd.make_dual(x.clone().requires_grad_(grad), torch.ones_like(x))
        for grad in (False, True):
            for call in (lambda: T.token_log_probs(dual(z, grad), y),
                         lambda: T.distillation(dual(z, grad), ids, t),
                         lambda: T.distillation_step(dual(z, grad), ids, t)):
                with pytest.raises(NativeError, match="forward-mode"):
                    call()


def test_tangents_of_gradients_are_refused(stand_in):
    import torch.autograd.forward_ad as fwd
    from defmuon_amd._native import NativeError
    T, _ = stand_in
    z, y, ids, t = _case()
    z, t = z.float().requires_grad_(), t.float()
    with fwd.dual_level():
        one = fwd.make_dual(torch.ones(5), torch.ones(5))
        for out in (T.token_log_probs(z, y).entropy, T.distillation(z, ids, t, reduction="none")):
            with pytest.raises(NativeError, match="forward-mode"):
                torch.autograd.grad(out, z, one)


@pytest.mark.filterwarnings("ignore")
def test_traces_record_the_call_or_refuse(stand_in):
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    from defmuon_amd._native import NativeError
    T, _ = stand_in
    z, y, ids, t = _case()
    z, t = z.float(), t.float()
    ops = (lambda x: T.token_log_probs(x * 2, y).log_probs,
           lambda x: T.token_log_probs(x * 2, y, top=2).top_log_probs,
           lambda x: T.distillation(x * 2, ids, t, reduction="none"))
    step = lambda x: T.distillation_step(x, ids, t)[1]   # noqa: E731
    for grad in (False, True):
        for op in ops:
            traced = torch.jit.trace(op, z.clone().requires_grad_(grad))
            assert torch.equal(traced(z + 1), op(z + 1))
    for op in (*ops, step):
        with pytest.raises(NativeError, match="trace"):
            make_fx(op)(z)
        with FakeTensorMode() as mode, pytest.raises(NativeError, match="trace"):
            op(mode.from_tensor(z))
    with pytest.raises(NativeError, match="trace"):
        torch.jit.trace(step, z)


def test_a_top_that_is_no_whole_number(stand_in):
    from defmuon_amd._native import NativeError
    T, _ = stand_in
    for top in (2.0, 2.5, None, "3"):
        with pytest.raises(NativeError, match="top"):
            T.token_log_probs(torch.randn(3, 9), top=top)


def test_a_temperature_that_is_no_number(stand_in):
    """A tensor's value would have to be waited for."""
    from defmuon_amd._native import NativeError
    T, _ = stand_in
    z, _, ids, t = _case()
    for tau in (torch.tensor(1.0), "1", None):
        with pytest.raises(NativeError, match="temperature"):
            T.token_log_probs(z.float(), temperature=tau)
        with pytest.raises(NativeError, match="temperature"):
            T.distillation(z.float(), ids, t.float(), temperature=tau)


def test_gradients_over_the_logits_are_refused(lib):
    """The gradient kernels read the listed classes' logits again behind their row's gradient."""
    z, other = ctypes.c_void_p(256), ctypes.c_void_p(4096)   # never read
    assert lib.dmh_log_probs_grad(None, z, 0, 2, 9, 9, other, 1, -100, 1.0, 3, other, other, other,
                                  None, other, z, 9) == 1
    assert b"dmh_log_probs_grad" in lib.dmh_last_error()
    assert lib.dmh_distill_grad(None, z, 0, 2, 9, 9, other, 1, 3, other, 0, -100, 1.0, other, None,
                                other, 0, z, 9) == 1
    assert b"dmh_distill_grad" in lib.dmh_last_error()
