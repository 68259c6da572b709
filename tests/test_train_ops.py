"""CPU checks of the training operators: the generator's published vectors, the host's checks
of arguments (no kernel is launched) and how tensors are taken as rows."""

import ctypes

import numpy as np
import pytest
import torch

import train_ref as R


# counter, key and result: the known-answer vectors published with the generator
@pytest.mark.parametrize("ctr,key,want", [
    ([0, 0, 0, 0], [0, 0], [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]),
    ([0xffffffff] * 4, [0xffffffff] * 2, [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]),
    ([0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344], [0xa4093822, 0x299f31d0],
     [0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1]),
])
def test_reference_generator_matches_its_published_vectors(ctr, key, want):
    got = R.philox(np.array([ctr[0] | ctr[1] << 32], dtype=np.uint64), key[0] | key[1] << 32,
                   ctr[2] | ctr[3] << 32)
    assert got[0].tolist() == want


def test_share_of_kept_elements():
    # binomial(2^20, 0.9): five standard deviations are 1536
    k = R.keep(0, 1 << 20, 0.1, (123, 4))
    assert abs(int(k.sum()) - 0.9 * (1 << 20)) < 1536
    assert torch.equal(k[24:1000], R.keep(24, 976, 0.1, (123, 4)))
    assert not torch.equal(k, R.keep(0, 1 << 20, 0.1, (123, 5)))


@pytest.fixture(scope="module")
def lib():
    from defmuon_amd import _native
    return _native.load()


def test_entry_points_refuse_without_launching(lib):
    one = ctypes.c_void_p(256)   # never read: every call below is refused on the host

    def drop(**kw):
        a = dict(x=one, xt=0, rows=2, cols=3, xs=3, res=None, rs=0, out=one, ot=0, cut=5)
        a.update(kw)
        return lib.dmh_dropout(None, a["x"], a["xt"], a["rows"], a["cols"], a["xs"], a["res"],
                               a["rs"], a["out"], a["ot"], a["cut"], 1, 2, None)
    for bad in (dict(xt=3), dict(ot=-1), dict(rows=-1), dict(cols=-1), dict(xs=-1), dict(rs=-3),
                dict(cut=-1), dict(cut=65537), dict(x=None), dict(out=None),
                dict(rows=1 << 40, cols=1 << 40)):
        assert drop(**bad) == 1, bad
        assert b"dmh_dropout" in lib.dmh_last_error()
    assert drop(rows=0, x=None) == 0 and drop(cols=0, out=None) == 0

    def embed(**kw):
        a = dict(ids=one, tokens=4, seq=2, w=one, dt=0, vocab=9, dim=8, ws=8, pw=None, pr=0,
                 ps=0, cut=0, out=one, ot=0)
        a.update(kw)
        return lib.dmh_embedding(None, a["ids"], 1, a["tokens"], a["seq"], a["w"], a["dt"],
                                 a["vocab"], a["dim"], a["ws"], a["pw"], a["pr"], a["ps"], None,
                                 1.0, a["cut"], 0, 0, None, a["out"], a["ot"])
    for bad in (dict(ids=None), dict(out=None), dict(w=None), dict(tokens=-1), dict(dim=-1),
                dict(vocab=-1), dict(dt=7), dict(ot=4), dict(cut=70000), dict(ws=-8),
                dict(pw=one, pr=2, ps=8, seq=0), dict(tokens=(1 << 40) + 1)):
        assert embed(**bad) == 1, bad
        assert b"dmh_embedding" in lib.dmh_last_error()
    assert embed(tokens=0, ids=None) == 0 and embed(dim=0, w=None) == 0

    def grad(**kw):
        a = dict(ids=one, pos=None, tokens=400, seq=2, g=one, dt=0, gs=8, rows=9, dim=8, cut=0,
                 out=one, pout=None, prows=0, ot=0, ws=one, nb=1 << 20)
        a.update(kw)
        return lib.dmh_embedding_grad(None, a["ids"], a["pos"], 1, a["tokens"], a["seq"], a["g"],
                                      a["dt"], a["gs"], a["dim"], -1, 1.0, a["cut"], 0, 0, None,
                                      a["out"], a["rows"], 0, a["pout"], a["prows"], 0, a["ot"],
                                      a["ws"], a["nb"])
    for bad in (dict(g=None), dict(ids=None), dict(tokens=-1), dict(tokens=1 << 27),
                dict(rows=-1), dict(rows=1 << 27), dict(dim=-1), dict(dim=1 << 30), dict(dt=9),
                dict(ot=9), dict(gs=-1), dict(cut=-2), dict(pout=one, prows=2, seq=0),
                dict(pout=one, prows=2, seq=3), dict(pout=one, prows=1 << 27)):
        assert grad(**bad) == 1, bad
        assert b"dmh_embedding_grad" in lib.dmh_last_error()
    assert grad(nb=3) == 2 and grad(ws=None) == 2
    assert b"workspace" in lib.dmh_last_error()
    assert grad(out=None) == 0 and grad(rows=0) == 0 and grad(dim=0) == 0

    nb = ctypes.c_size_t()
    size = lib.dmh_embedding_grad_workspace_size
    assert size(-1, 5, 5, 8, 0, ctypes.byref(nb)) == 1 and size(5, 5, 5, 8, 0, None) == 1
    assert size(5, 1 << 27, 5, 8, 0, ctypes.byref(nb)) == 1
    assert size(1000, 0, 0, 8, 1, ctypes.byref(nb)) == 0 and nb.value == 0
    # sorted tokens and parts of 32 chunks; implicit positions have parts alone
    assert size(1000, 50, 0, 64, 0, ctypes.byref(nb)) == 0
    assert nb.value == 2 * 4096 + 32 * 2 * 64 * 4
    assert size(1000, 0, 50, 64, 0, ctypes.byref(nb)) == 0 and nb.value == 32 * 2 * 64 * 4

    def xent(**kw):
        a = dict(z=one, dt=0, rows=2, v=5, zs=5, y=one, red=1, loss=one, count=one, ds=5, ws=one,
                 nb=1 << 20)
        a.update(kw)
        return lib.dmh_cross_entropy(None, a["z"], a["dt"], a["rows"], a["v"], a["zs"], a["y"], 1,
                                     -100, 0.0, 0.0, a["red"], 1.0, a["loss"], a["count"], None,
                                     None, a["ds"], a["ws"], a["nb"])
    for bad in (dict(z=None), dict(y=None), dict(loss=None), dict(count=None), dict(dt=3),
                dict(rows=-1), dict(rows=1 << 22), dict(v=0), dict(v=1 << 31), dict(zs=-1),
                dict(ds=-1), dict(red=3), dict(red=-1)):
        assert xent(**bad) == 1, bad
        assert b"dmh_cross_entropy" in lib.dmh_last_error()
    assert xent(ws=None) == 2 and xent(nb=1) == 2
    assert xent(rows=0, red=0) == 0

    def xgrad(**kw):
        a = dict(z=one, dt=0, rows=2, v=5, zs=5, y=one, lse=one, go=one, dz=one, ds=5)
        a.update(kw)
        return lib.dmh_cross_entropy_grad(None, a["z"], a["dt"], a["rows"], a["v"], a["zs"],
                                          a["y"], 1, -100, 0.0, 0.0, a["lse"], None, a["go"], 0,
                                          a["dz"], a["ds"])
    for bad in (dict(z=None), dict(y=None), dict(lse=None), dict(go=None), dict(dz=None),
                dict(dt=5), dict(rows=1 << 22), dict(v=0), dict(zs=-2), dict(ds=-2)):
        assert xgrad(**bad) == 1, bad
        assert b"dmh_cross_entropy_grad" in lib.dmh_last_error()
    assert xgrad(rows=0) == 0
    assert lib.dmh_cross_entropy_workspace_size(1, 0, ctypes.byref(nb)) == 1
    assert lib.dmh_cross_entropy_workspace_size(1, 1, None) == 1


def test_no_cpu_fallback():
    from defmuon_amd import train_ops as T
    from defmuon_amd._native import NativeError
    x, ids = torch.randn(4, 8), torch.zeros(4, dtype=torch.int64)
    for call in (lambda: T.dropout(x, 0.1, (1, 2)), lambda: T.dropout_backward(x, 0.1, (1, 2)),
                 lambda: T.embedding(ids, x), lambda: T.embedding_backward(x, ids, 5),
                 lambda: T.cross_entropy(x, ids), lambda: T.cross_entropy_step(x, ids)):
        with pytest.raises(NativeError, match="GPU"):
            call()
    with pytest.raises(NativeError):
        T.Dropout(1.5)
    assert T.Dropout(0.3).eval()(x) is x


def test_tensors_as_rows():
    from defmuon_amd.train_ops import _rows
    x = torch.arange(240.0).view(4, 5, 12)
    for t, rows, stride, same in [
            (x, 20, 12, True), (x[..., :7], 20, 12, True), (x[:, ::2], 12, 24, False),
            (x[:, 1:2, 3:], 4, 60, True), (x[::2, :, 1:], 10, 12, False),
            (x.transpose(0, 1), 20, 12, False), (x.mT, 48, 5, False),
            (x[0, 0].expand(4, 5, 12), 20, 0, True), (x[:1, :1], 1, 12, True),
            (torch.ones(()).expand(3, 4), 3, 4, False), (x[..., 3:4], 20, 12, True)]:
        r, n, cols, st = _rows(t)
        assert (n, cols) == (rows, t.shape[-1])
        assert (r is t) == same
        want = t.reshape(-1, cols)
        flat = torch.as_strided(r, (n, cols), (st, 1), r.storage_offset())
        assert torch.equal(flat, want)
    assert _rows(torch.empty(0, 3))[1:] == (0, 3, 3)
    assert _rows(torch.empty(3, 0))[1] == 0


def test_draws_follow_the_seed():
    from defmuon_amd.train_ops import draw_rng
    torch.manual_seed(3)
    a, b = draw_rng(), draw_rng()
    torch.manual_seed(3)
    assert draw_rng() == a != b


@pytest.fixture
def stand_in(monkeypatch):
    """train_ops on CPU tensors: plain forms in place of the launches."""
    from defmuon_amd import _native, train_ops as T

    def cross_entropy(z, rows, y, ignore, smoothing, z_loss, reduction, grad_scale, loss, dz,
                      dstride, keep):
        assert all(type(n) is int for n in rows)
        zz = z.detach().clone()
        rows, d, _ = R.xent(zz, y, ignore, smoothing, z_loss)
        n = 1 if reduction == 2 else int((y != ignore).sum())
        loss.copy_(rows if reduction == 0 else rows.sum() / n)
        if dz is not None:   # through its memory, as a kernel writes it
            dz.numpy()[...] = (d * grad_scale / n).float().numpy()
        return torch.zeros(1)

    def embedding_grad(ids, positions, tokens, seq, grad, stride, dim, padding, scale, cut, rng,
                       out, add, pos_out, pos_add):
        for table in (out, pos_out):
            if table is not None:
                table.numpy()[...] += 1.0

    monkeypatch.setattr(T, "_float", lambda *a: None)
    monkeypatch.setattr(_native, "cross_entropy", cross_entropy)
    monkeypatch.setattr(_native, "embedding_grad", embedding_grad)
    return T


def test_writes_in_place_are_seen_by_autograd(stand_in):
    T = stand_in
    h, y = torch.randn(6, 11, requires_grad=True), torch.arange(6)
    w = torch.randn(11, 11)
    want = {}
    for name, f in (("tanh", torch.tanh), ("product", lambda t: t @ w)):
        z = f(h)
        (want[name],) = torch.autograd.grad(z, h, T.cross_entropy_step(z, y)[1])
        assert z._version == 0
    z = h @ w   # its backward pass needs no logits
    loss, dz = T.cross_entropy_step(z, y, inplace=True)
    assert dz.data_ptr() == z.data_ptr() and z._version == 1
    assert torch.equal(torch.autograd.grad(z, h, dz)[0], want["product"])
    for view in (lambda t: t.view(2, 3, 11), lambda t: t[:, :9]):   # ... nor has it as a view
        z = view(h @ w)
        t = y.clamp(max=8).view(z.shape[:-1])
        ref = torch.autograd.grad(z, h, T.cross_entropy_step(z, t)[1], retain_graph=True)[0]
        assert torch.equal(torch.autograd.grad(z, h, T.cross_entropy_step(z, t, inplace=True)[1])[0],
                           ref)
    z = torch.tanh(h)
    dz = T.cross_entropy_step(z, y, inplace=True)[1]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward(dz)
    z = h @ w   # a loss that has saved the same logits
    loss = T.cross_entropy(z, y)
    T.cross_entropy_step(z, y, inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        T.cross_entropy_step(h @ w, y, inplace=True)
    g, ids = torch.randn(2, 3, 8), torch.zeros(2, 3, dtype=torch.int64)
    dw, dp = torch.zeros(5, 8), torch.zeros(4, 8)
    T.embedding_backward(g, ids, 5, pos_rows=4, weight_grad=dw)
    assert (dw._version, dp._version) == (1, 0) and bool((dw == 1).all())
    T.embedding_backward(g, ids, 5, pos_rows=4, weight_grad=dw, pos_grad=dp)
    assert (dw._version, dp._version) == (2, 1)


def test_entries_that_keep_row_statistics_refuse(lib):
    one = ctypes.c_void_p(256)   # never read

    def fwd(top=one, total=one, rows=2, dt=0, red=1):
        return lib.dmh_cross_entropy_stats(None, one, dt, rows, 5, 5, one, 1, -100, 0.0, 0.0, red,
                                           1.0, one, one, top, total, None, 5, one, 1 << 20)

    def bwd(top=one, total=one, rows=2, dt=0):
        return lib.dmh_cross_entropy_grad_stats(None, one, dt, rows, 5, 5, one, 1, -100, 0.0, 0.0,
                                                top, total, None, one, 0, one, 5)
    for call in (fwd, bwd):
        for bad in (dict(top=None), dict(total=None), dict(rows=1 << 22), dict(dt=3)):
            assert call(**bad) == 1, bad
            assert b"dmh_cross_entropy" in lib.dmh_last_error()
    assert fwd(rows=0, red=0, top=None, total=None) == 0 and bwd(rows=0, total=None) == 0


@pytest.mark.filterwarnings("ignore::DeprecationWarning")
def test_forward_mode_is_refused(monkeypatch):
    """A tangent is never dropped, whether or not a gradient is wanted too."""
    import torch.autograd.forward_ad as fwd
    from defmuon_amd import train_ops as T
    from defmuon_amd._native import NativeError
    w, x = torch.randn(4, 8), torch.randn(2, 3, 8)
    ids = torch.zeros(2, 3, dtype=torch.int64)
    with fwd.dual_level():
        def dual(t, grad=False):
            return fwd.make_dual(t.clone().requires_grad_(grad), torch.ones_like(t))
        for grad in (False, True):
            for call in (lambda: T.dropout(dual(x, grad), 0.1, (1, 2)),
                         lambda: T.dropout_backward(dual(x, grad), 0.1, (1, 2)),
                         lambda: T.embedding(ids, dual(w, grad)),
                         lambda: T.embedding_backward(dual(x, grad), ids, 4),
                         lambda: T.cross_entropy(dual(x, grad), ids),
                         lambda: T.cross_entropy_step(dual(x, grad), ids)):
                with pytest.raises(NativeError, match="forward-mode"):
                    call()
        with pytest.raises(NativeError, match="GPU"):   # without a tangent, the ordinary way
            T.dropout(x, 0.1, (1, 2))
        monkeypatch.setattr(T, "_float", lambda *a: None)   # past the first table's check
        with pytest.raises(NativeError, match="forward-mode"):
            T.embedding(ids, w, dual(w))


def test_a_tangent_of_the_gradient_is_refused(stand_in):
    import torch.autograd.forward_ad as fwd
    from defmuon_amd._native import NativeError
    z = torch.randn(6, 11, requires_grad=True)
    with fwd.dual_level():
        loss = stand_in.cross_entropy(z, torch.arange(6))
        with pytest.raises(NativeError, match="forward-mode"):
            torch.autograd.grad(loss, z, fwd.make_dual(torch.ones(()), torch.ones(())))


@pytest.mark.filterwarnings("ignore")
def test_traces_record_the_call_or_refuse(stand_in, monkeypatch):
    """torch.jit.trace records autograd functions; every other trace would hold the allocation
    of the results alone."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils.flop_counter import FlopCounterMode
    from defmuon_amd import _native
    T = stand_in

    def dropout(x, residual, out, cut, rng, rows):
        out.detach().numpy()[...] = 2 * x.detach().numpy()

    def embedding(ids, weight, pos_weight, positions, scale, cut, rng, out):
        out.detach().numpy()[...] = weight.detach().numpy()[ids.numpy()]
    monkeypatch.setattr(_native, "dropout", dropout)
    monkeypatch.setattr(_native, "embedding", embedding)
    x, z, y = torch.randn(3, 5), torch.randn(3, 5), torch.arange(3)
    ops = (lambda t: T.dropout(t + 1, 0.1, (1, 2)) * 3, lambda t: T.embedding(y, t),
           lambda t: T.cross_entropy(t, y, reduction="none"))
    steps = (lambda t: T.dropout_backward(t, 0.1, (1, 2)),
             lambda t: T.embedding_backward(t, y, 4)[0], lambda t: T.cross_entropy_step(t, y)[1])
    for grad in (False, True):
        for op in ops:
            traced = torch.jit.trace(op, x.clone().requires_grad_(grad))
            assert torch.equal(traced(z), op(z))
    for op in ops + steps:
        for kw in ({}, dict(tracing_mode="symbolic"), dict(pre_dispatch=True)):
            with pytest.raises(_native.NativeError, match="trace"):
                make_fx(op, **kw)(x)
        with FakeTensorMode() as mode, pytest.raises(_native.NativeError, match="trace"):
            op(mode.from_tensor(x))
        with FlopCounterMode(display=False):   # a mode that records nothing
            op(x)
    for op in steps:
        with pytest.raises(_native.NativeError, match="trace"):
            torch.jit.trace(op, x)


def test_positions_and_ids_keep_their_values():
    from defmuon_amd.train_ops import _positions
    a, b = torch.tensor([3, -1], dtype=torch.int32), torch.tensor([2 ** 32 + 1, -2 ** 32])
    for ids, positions, dtype in ((a, b, torch.int64), (b, a, torch.int64),
                                  (a, a.flip(0), torch.int32), (b, b.flip(0), torch.int64)):
        i, p = _positions(positions, ids, "embedding")
        assert i.dtype == p.dtype == dtype
        assert i.tolist() == ids.tolist() and p.tolist() == positions.tolist()
    assert _positions(None, a, "embedding")[0] is a


def test_draws_come_from_the_cpu_generator():
    from defmuon_amd.train_ops import draw_rng
    torch.manual_seed(3)
    want = draw_rng()
    torch.manual_seed(3)
    with torch.device("meta"):   # a default device for the program's own tensors
        assert draw_rng() == want


def test_graphs_and_traces_do_not_repeat_a_mask(monkeypatch):
    from defmuon_amd import train_ops as T
    from defmuon_amd._native import NativeError
    x = torch.randn(4, 8)
    monkeypatch.setattr(T, "dropout", lambda x, p, rng, residual: rng)
    m, state = T.Dropout(0.3), torch.zeros(5, 2, dtype=torch.int64)
    assert m(x) != m(x) and m(x, rng=(1, 2)) == (1, 2) and m(x, rng=state[3]).tolist() == [0, 0]
    with monkeypatch.context() as c:
        c.setattr(torch.cuda, "is_initialized", lambda: True)
        c.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        for call in (T.draw_rng, lambda: m(x)):
            with pytest.raises(NativeError, match="graph"):
                call()
        assert m(x, rng=state[1]).tolist() == [0, 0]   # not drawn here
        assert m.eval()(x) is x and m(x, residual=x) is None
    with pytest.raises(NativeError, match="trace"), pytest.warns():
        torch.jit.trace(lambda t: t * T.draw_rng()[0], x)


def test_an_rng_tensor_changed_before_the_backward_pass(stand_in, monkeypatch):
    from defmuon_amd import _native
    T, seen = stand_in, []
    monkeypatch.setattr(_native, "dropout", lambda *a: seen.append(a[4]))
    monkeypatch.setattr(_native, "embedding", lambda *a: None)
    x = torch.randn(3, 8, requires_grad=True)
    state, ids = torch.tensor([[1, 2], [1, 3]]), torch.zeros(2, 3, dtype=torch.int64)
    for op in (lambda rng: T.dropout(x, 0.5, rng), lambda rng: T.dropout(x, 0.5, rng, residual=x),
               lambda rng: T.embedding(ids, x, dropout_p=0.5, rng=rng)):
        op(state[1]).sum().backward()
        op((5, 6)).sum().backward()
        y = op(state[1])
        state[:, 0] += 1
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
    assert seen[1] == (0, 0, state[1].data_ptr()) and seen[3] == (5, 6, 0)


def test_the_workspace_is_the_librarys_size(monkeypatch):
    """The allocation and the size passed follow dmh_cross_entropy_workspace_size."""
    from defmuon_amd import _native
    seen = []

    class Lib:
        def dmh_cross_entropy_workspace_size(self, rows, classes, out):
            out._obj.value = 1000 * rows + classes
            return 0

        def dmh_cross_entropy_stats(self, *a):
            seen.append(a)
            return 0
    _native.cross_entropy_workspace_bytes.cache_clear()
    monkeypatch.setattr(_native, "_lib", Lib())
    monkeypatch.setattr(_native, "_raw_stream", lambda index: 0)
    monkeypatch.setattr(_native, "_current_device", lambda: -1)
    z, y = torch.randn(3, 5), torch.arange(3)
    stats = _native.cross_entropy(z, (3, 5, 5), y, -100, 0.0, 0.0, 1, 1.0, torch.empty(()), None, 0)
    _native.cross_entropy_workspace_bytes.cache_clear()
    at, nbytes = seen[0][-2:]
    assert nbytes == 3005
    assert stats.data_ptr() + 4 * stats.numel() >= at + nbytes


def test_rows_of_more_columns_than_an_int_counts(lib, monkeypatch):
    """A C int would keep the low 32 bits of the width."""
    from defmuon_amd import _native, train_ops as T
    one = ctypes.c_void_p(256)   # never read
    assert lib.dmh_embedding(None, one, 1, 1, 1, one, 0, 2, (1 << 30) + 1, 8, None, 0, 0, None, 1.0,
                             0, 0, 0, None, one, 0) == 1
    monkeypatch.setattr(T, "_float", lambda *a: None)
    for name in ("embedding", "embedding_grad"):
        monkeypatch.setattr(_native, name, lambda *a: pytest.fail("launched"))
    x, ids = torch.zeros(()), torch.zeros(1, dtype=torch.int64)
    for wide in ((1 << 30) + 1, (1 << 32) + 8):
        with pytest.raises(_native.NativeError, match="too long"):
            T.embedding(ids, x.expand(2, wide))
        with pytest.raises(_native.NativeError, match="too long"):
            T.embedding_backward(x.expand(1, wide), ids, 2)
    with pytest.raises(_native.NativeError, match="too long"):
        T.embedding(ids.expand((1 << 32) + 1), x.expand(2, 8), x.expand(1 << 33, 8))


def test_tensors_without_memory_do_not_pass_for_absent_ones(monkeypatch):
    from defmuon_amd import _native as N

    class Wrapper(torch.Tensor):
        """As a distributed tensor: no storage of its own."""
        @staticmethod
        def __new__(cls, t):
            return torch.Tensor._make_wrapper_subclass(cls, t.shape, dtype=t.dtype,
                                                       device=t.device, strides=t.stride())

        __torch_dispatch__ = classmethod(lambda *a, **kw: pytest.fail("dispatched"))
    monkeypatch.setattr(N, "_lib", type("Lib", (), {"__getattr__": lambda *a: lambda *b: 0})())
    monkeypatch.setattr(N, "_raw_stream", lambda index: 0)
    monkeypatch.setattr(N, "_current_device", lambda: -1)
    x, ids, rng = torch.randn(3, 8), torch.zeros(3, dtype=torch.int64), (0, 0, 0)

    def grad(positions, out, pos_out):
        N.embedding_grad(ids, positions, 3, 3, x, 8, 8, -1, 1.0, 0, rng, out, True, pos_out, True)

    def embed(pos, positions):
        N.embedding(ids, x, pos, positions, 1.0, 0, rng, torch.empty(3, 8))
    N.dropout(x, x, x, 0, rng, (3, 8, 8, 8))   # the stand-in takes ordinary tensors
    embed(x, ids), grad(ids, x, x)
    embed(torch.empty(0, 8), ids)
    w = Wrapper(x)
    for call in (lambda: N.dropout(x, w, x, 0, rng, (3, 8, 8, 8)), lambda: embed(w, None),
                 lambda: embed(x, Wrapper(ids)), lambda: grad(Wrapper(ids), x, x),
                 lambda: grad(None, w, None), lambda: grad(None, None, w)):
        with pytest.raises(N.NativeError, match="no memory"):
            call()
    N.embedding_grad_workspace_bytes.cache_clear()
