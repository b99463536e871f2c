"""The causal mixer's operators in 64 bits, from their formulas, with bounds of what fp32 arithmetic may be off by.

Gradients are autograd's of these functions.  `U` is fp32's half step, 2^-24; outputs add half a step of their own type (`half_step`)."""
import torch

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def silu(x):
    return x * torch.sigmoid(x)


def inside(lengths, B, L, device):
    if lengths is None:
        return torch.ones(B, L, 1, dtype=torch.bool, device=device)
    return (torch.arange(L, device=device) < lengths.unsqueeze(1)).unsqueeze(-1)


def conv(x, w, bias=None, act=None, state=None, lengths=None):
    """-> (y, state behind the last position)"""
    B, L, C = x.shape
    K = w.shape[1]
    ok = inside(lengths, B, L, x.device)
    before = torch.zeros(B, K - 1, C, dtype=x.dtype, device=x.device) if state is None else state
    rows = torch.cat([before, torch.where(ok, x, torch.zeros_like(x))], 1)
    pre = torch.zeros_like(x) if bias is None else bias.expand(B, L, C)
    for k in range(K):
        pre = pre + w[:, k] * rows[:, k:k + L]
    y = silu(pre) if act == "silu" else pre
    y = torch.where(ok, y, torch.zeros_like(y))
    ends = [L] * B if lengths is None else [min(max(int(n), 0), L) for n in lengths]
    return y, torch.stack([rows[b, n:n + K - 1] for b, n in enumerate(ends)])


def scan(x, dt, A, Bm, Cm, D=None, z=None, dt_bias=None, softplus=False, state=None, lengths=None):
    """-> (y, state behind the last position)"""
    B, L, C = x.shape
    if Bm.dim() == 3:
        Bm, Cm = Bm.unsqueeze(2), Cm.unsqueeze(2)
    each = C // Bm.shape[2]
    ok = inside(lengths, B, L, x.device)
    d = dt if dt_bias is None else dt + dt_bias
    if softplus:
        d = torch.logaddexp(d, torch.zeros_like(d))
    d = torch.where(ok, d, torch.zeros_like(d))
    x = torch.where(ok, x, torch.zeros_like(x))
    h = torch.zeros(B, C, A.shape[1], dtype=x.dtype, device=x.device) if state is None else state
    ys = []
    for t in range(L):
        b, c = (m[:, t].repeat_interleave(each, 1) for m in (Bm, Cm))
        h = torch.exp(d[:, t, :, None] * A) * h + (d[:, t] * x[:, t]).unsqueeze(-1) * b
        ys.append((h * c).sum(-1))
    y = torch.stack(ys, 1)
    if D is not None:
        y = y + D * x
    if z is not None:
        y = y * silu(z)
    return torch.where(ok, y, torch.zeros_like(y)), h


def norm(x, groups, w=None, b=None, eps=1e-5, act=None):
    N, C = x.shape[0], x.shape[-1]
    v = x.reshape(N, -1, groups, C // groups)
    v = v - v.mean((1, 3), keepdim=True)
    v = (v / torch.sqrt((v * v).mean((1, 3), keepdim=True) + eps)).reshape(x.shape)
    if w is not None:
        v = v * w
    if b is not None:
        v = v + b
    if act == "silu":
        return silu(v)
    return v * torch.special.ndtr(v) if act == "gelu" else v


def doubles(ins, grad=True):
    """Copies in 64 bits, leaves of a graph where they are numbers."""
    return {k: None if t is None else t.detach().double().requires_grad_(grad) if t.is_floating_point() else t for k, t in ins.items()}


def within(name, got, want, bound):
    """|got - want| <= bound + half a step of got's type, everywhere.  Below fp32's normal numbers a factor (a decay exp(-90), say) may come out as 0 and so be off by all of itself, up to 2^-126; what
    multiplies it in these tests (states, inputs and sums of 256 of them) stays below 2^16, so 2^-110 is added.  A bound is at least U times the magnitudes that a sum is made of: where bound / U
    passes 2^127, partial sums may pass fp32's range (decays above 1, from steps below 0), and nothing is said of the result."""
    assert got.shape == want.shape, (name, got.shape, want.shape)
    bound = torch.as_tensor(bound, dtype=torch.float64, device=got.device).expand(got.shape)
    fits = bound / U < 2.0 ** 127
    got, want, bound = got[fits], want[fits], bound[fits]
    off = (got.double() - want).abs()
    room = bound + half_step(got.dtype) * want.abs() + 2.0 ** -110
    worst = (off - room).max().item() if off.numel() else -1
    assert torch.isfinite(got).all() and worst <= 0, f"{name}: off by {off.max().item():.3g}, {(off / room).max().item():.3g} times what is allowed"
