"""Plain 64-bit forms of dropout, the linear layer and the loss head, for the tests."""
import numpy as np
import torch

LOW = 0xFFFFFFFF


def philox(ctr, key):
    """Philox4x32-10 of Salmon et al. (SC 2011) on uint64 arrays holding 32-bit words."""
    c, (k0, k1) = [np.asarray(v, dtype=np.uint64) for v in ctr], key
    s, low = np.uint64(32), np.uint64(LOW)
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> s) ^ c[1] ^ np.uint64(k0), b & low, (a >> s) ^ c[3] ^ np.uint64(k1), a & low]
        k0, k1 = (k0 + 0x9E3779B9) & LOW, (k1 + 0xBB67AE85) & LOW
    return c


def keep_mask(seed, offset, rows, cols, p):
    """(mask [rows, cols] bool, scale): element (r, c) compares 16-bit lane c % 8 at counter
    (c / 8, r, offset) with round(p 65536)."""
    n8 = (cols + 7) // 8
    seed, offset = seed & (2**64 - 1), offset & (2**64 - 1)
    one = np.ones((rows, n8), dtype=np.uint64)
    words = philox([one * np.arange(n8, dtype=np.uint64),
                    one * np.arange(rows, dtype=np.uint64)[:, None],
                    one * np.uint64(offset & LOW), one * np.uint64(offset >> 32)],
                   (seed & LOW, seed >> 32))
    lanes = np.stack([(w >> np.uint64(16 * h)) & np.uint64(0xFFFF) for w in words for h in (0, 1)], -1)
    t = int(round(float(np.float32(p)) * 65536))
    keep = lanes.reshape(rows, n8 * 8)[:, :cols].astype(np.int64) >= t
    return torch.from_numpy(keep), (65536.0 / (65536 - t) if t < 65536 else 0.0)


def act(z, name):
    if name == "relu":
        return z.clamp(min=0)
    if name == "gelu":
        return z * torch.sigmoid(2 * 0.7978845608 * (z + 0.044715 * z ** 3))
    return z * torch.sigmoid(z) if name == "silu" else z


def act_grad(z, name):
    z = z.detach().requires_grad_(True)
    g, = torch.autograd.grad(act(z, name).sum(), z)
    return (z > 0).to(z.dtype) if name == "relu" else g


def sigmoid_arg(z, name):
    """The argument of the sigmoid inside an activation (its error grows with it)."""
    return 2 * 0.7978845608 * (z + 0.044715 * z ** 3) if name == "gelu" else z


def head(x, w, targets, smoothing):
    """(row losses, lse, logits, target distribution, valid) for w [V, C]."""
    V = w.shape[0]
    z = x @ w.t()
    lse = torch.logsumexp(z, 1)
    valid = (targets >= 0) & (targets < V)
    t = targets.long().clamp(0, V - 1)
    y = torch.full_like(z, smoothing / (V - 1) if V > 1 else 0.0)
    # one class alone: y sums to 1, since a constant loss has no gradient
    y.scatter_(1, t[:, None], 1.0 - smoothing if V > 1 else 1.0)
    loss = (y * (lse[:, None] - z)).sum(1)
    return torch.where(valid, loss, torch.zeros_like(loss)), lse, z, y, valid
