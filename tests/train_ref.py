"""Plain 64-bit forms of the training operators, on the CPU, and their error bounds."""

import numpy as np
import torch

# unit roundoff of a result's type; fp32 arithmetic inside
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}
E32 = 2.0 ** -24


def philox(blocks, seed, offset):
    """Philox4x32-10 words (n, 4) uint32 of the blocks (counter low half), key seed."""
    b = np.asarray(blocks, dtype=np.uint64)
    m32, s32 = np.uint64(0xFFFFFFFF), np.uint64(32)
    c = [b & m32, b >> s32, np.full_like(b, offset & 0xFFFFFFFF), np.full_like(b, offset >> 32)]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        a, d = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(d >> s32) ^ c[1] ^ np.uint64(k[0]), d & m32,
             (a >> s32) ^ c[3] ^ np.uint64(k[1]), a & m32]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, axis=1).astype("<u4")


def keep(first, count, p, rng):
    """Kept elements (bool tensor) among flat indices first .. first + count - 1."""
    cut = int(round(p * 65536))
    b0, b1 = first // 8, (first + count + 7) // 8
    mod = (1 << 64) - 1
    draws = philox(np.arange(b0, b1), rng[0] & mod, rng[1] & mod).view("<u2").reshape(-1)
    return torch.from_numpy(draws[first - 8 * b0:][:count].astype(np.int32) >= cut)


def drop_scale(p):
    cut = int(round(p * 65536))
    return 65536.0 / (65536 - cut) if cut < 65536 else 0.0


def drop(x, p, rng):
    """Dropout of a float64 tensor."""
    if int(round(p * 65536)) == 0:
        return x
    k = keep(0, x.numel(), p, rng).view(x.shape)
    return torch.where(k, x * drop_scale(p), torch.zeros((), dtype=torch.float64))


def embedding(ids, w, pos=None, positions=None, scale=1.0, p=0.0, rng=None):
    x = w.double()[ids.long()] * scale
    if pos is not None:
        t = torch.arange(ids.shape[-1]).expand(ids.shape) if positions is None else positions
        x = x + pos.double()[t.long()]
    return drop(x, p, rng)


def table_grad(g, ids, rows, scale=1.0, p=0.0, rng=None, padding=None):
    """(gradient, sum of magnitudes, terms) of a table, each by row."""
    d = drop(g.double(), p, rng).reshape(-1, g.shape[-1])
    idx = ids.reshape(-1).long()
    ok = (idx >= 0) & (idx < rows)
    if padding is not None:
        ok &= idx != padding
    d, idx = d[ok], idx[ok]
    z = torch.zeros(rows, g.shape[-1], dtype=torch.float64)
    n = torch.zeros(rows, dtype=torch.float64).index_add_(0, idx, torch.ones(len(idx)).double())
    return (z.clone().index_add_(0, idx, d) * scale,
            z.clone().index_add_(0, idx, d.abs()) * abs(scale), n[:, None])


def xent(z, y, ignore=-100, eps=0.0, zeta=0.0):
    """(row losses, d loss_row / d z, lse) in float64; ignored rows are zero."""
    z = z.double()
    v = z.shape[-1]
    live = y != ignore
    t = torch.where(live, y, torch.zeros_like(y)).long()
    lse = torch.logsumexp(z, -1)
    zy = z.gather(-1, t[..., None])[..., 0]
    loss = lse - (1 - eps) * zy + zeta * lse * lse
    if eps:
        loss = loss - eps * z.mean(-1)
    q = torch.zeros_like(z).scatter_(-1, t[..., None], 1 - eps) + eps / v
    dz = torch.exp(z - lse[..., None]) * (1 + 2 * zeta * lse[..., None]) - q
    zero = torch.zeros((), dtype=torch.float64)
    return torch.where(live, loss, zero), torch.where(live[..., None], dz, zero), lse


def close(got, want, bound, what=""):
    """Every element of got within bound of want; NaN and infinities where want has them."""
    got, want = got.detach().cpu().double(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    odd = ~torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    assert torch.equal(got[odd & ~torch.isnan(want)], want[odd & ~torch.isnan(want)]), what
    bound = torch.as_tensor(bound, dtype=torch.float64).expand(want.shape)
    err = (got - want).abs()
    bad = ~odd & ~(err <= bound)
    assert not bad.any(), (what, float(err[bad].max()), float(bound[bad].min()),
                           int(bad.sum()), torch.nonzero(bad)[:4].tolist())
