"""Plain 64-bit forms of the operators of lvd_pg_b200/heads.py and bounds on what fp32 kernels may be off by.

Bounds, in units of u = 2^-24 (half a step of fp32 at one).  With d = (x - max) log2(e) / T: a difference, its product with
a rounded constant: d is off by 3 u |d|, so 2^d relatively by 3 u |d| ln2, and by 4 u for the exponential itself (2 ulp).
Sums: one u per addition in a chain of at most `chain`.  Hence, with D = sum p |d|,
  S relatively by u (4 + 3 D + chain), ln S absolutely by that and 2 u |ln S|; logp further 4 u |x_t - max| / T and u |logp|;
  A = sum 2^d d: each term u (4 + 3 + 3 |d|) of itself, the sum chain: u ((7 + chain) D + 3 D2), D2 = sum p d^2.
They are doubled for what the joining of partial sums adds."""
import numpy as np
import torch

U = 2.0 ** -24
LOG2E = 1.4426950408889634


def chain_of(cats):
    return cats / 64 + 64


class Logprobs:
    """log-probabilities, entropy and alternatives of x [rows, cats], and the bounds of the first two."""

    def __init__(self, x, tokens, top_k, temperature):
        x = x.detach().double()
        self.x, self.T, cats = x, temperature, x.shape[1]
        m = x.amax(1, keepdim=True)
        shift = torch.where(m == -np.inf, torch.zeros_like(m), m)
        e = ((x - shift) / temperature).exp()
        S = e.sum(1, keepdim=True)
        empty = S == 0
        self.empty = empty[:, 0]
        lnS = torch.where(empty, torch.ones_like(S), S).log()
        self.logp_all = (x - shift) / temperature - lnS
        self.p = e / torch.where(empty, torch.ones_like(S), S)
        pl = torch.where(self.p > 0, self.p * self.logp_all, torch.zeros_like(self.p))
        self.entropy = -pl.sum(1)
        d = torch.where(self.p > 0, (x - shift).abs() * LOG2E / temperature, torch.zeros_like(x))
        self.d, self.D, D2 = d, (self.p * d).sum(1), (self.p * d * d).sum(1)
        c = chain_of(cats)
        self.tol_S = 2 * U * (4 + 3 * self.D + c)
        lnS = lnS[:, 0]
        self.lnS = lnS.abs()
        self.tol_logp_all = (self.tol_S + 4 * U * self.lnS)[:, None] + 4 * U * (x - shift).abs() / temperature + 2 * U * self.logp_all.abs()
        self.tol_entropy = self.tol_S + 4 * U * self.lnS + 2 * U * ((11 + 2 * c) * self.D + 3 * D2 + 6 * self.D ** 2) + 2 * U * self.entropy.abs()
        if tokens is not None:
            t = tokens.long()
            given = (t >= 0) & (t < cats)
            at = torch.where(given, t, torch.zeros_like(t))[:, None]
            self.given, self.at = given, at
            self.logp = self.logp_all.gather(1, at)[:, 0]
            self.logp = torch.where(t < 0, torch.zeros_like(self.logp), torch.where(t >= cats, torch.full_like(self.logp, np.nan), self.logp))
            self.tol_logp = torch.where(given, self.tol_logp_all.gather(1, at)[:, 0], torch.full_like(self.logp, 0.0))
        order = np.lexsort((np.arange(cats)[None, :].repeat(x.shape[0], 0), -np.nan_to_num(x.cpu().numpy(), nan=np.inf, posinf=np.inf, neginf=-np.inf)))
        self.top_ids = torch.from_numpy(order[:, :top_k].copy()).to(x.device)
        self.top_logp = self.logp_all.gather(1, self.top_ids)
        self.tol_top = self.tol_logp_all.gather(1, self.top_ids)

    def grad(self, g_logp, g_entropy, g_top, dtype):
        """(gradient, bound): dx = (gL ([t] - p) + sum gK ([id] - p) - gH p (logp + H)) / T.  p is off relatively by
        u (4 + 3 |d|) and what S is; the factor of p is a sum of `terms` whose cancellation the bound does not use."""
        zero = torch.zeros(self.x.shape[0], dtype=torch.float64, device=self.x.device)
        gl = zero if g_logp is None else torch.where(self.given, g_logp.double(), zero)
        gh = zero if g_entropy is None else g_entropy.double()
        gk = torch.zeros_like(self.top_logp) if g_top is None else g_top.double()
        logp = torch.where(self.p > 0, self.logp_all, torch.zeros_like(self.p))
        total = gl + gk.sum(1)
        dx = -self.p * (total[:, None] + gh[:, None] * (logp + self.entropy[:, None]))
        weight = (gl.abs() + gk.abs().sum(1) + gh.abs() * (self.entropy + self.lnS))[:, None] + gh.abs()[:, None] * self.d
        tol = self.p * weight * (U * (24 + gk.shape[1] + 8 * self.d) + 2 * self.tol_S[:, None]) + self.p * (gh.abs() * self.tol_entropy)[:, None]
        pointed = torch.zeros_like(dx)
        if g_logp is not None:
            pointed.scatter_add_(1, self.at, gl[:, None])
        if g_top is not None:
            pointed.scatter_add_(1, self.top_ids, gk)
        spread = torch.zeros_like(dx)
        if g_logp is not None:
            spread.scatter_add_(1, self.at, gl.abs()[:, None])
        if g_top is not None:
            spread.scatter_add_(1, self.top_ids, gk.abs())
        dx = torch.where(self.empty[:, None], torch.zeros_like(dx), dx + pointed) / self.T
        tol = (tol + 40 * U * spread + 2.0 ** -118 * weight) / self.T
        return dx, tol + rounding(dx, dtype)


def rounding(value, dtype):
    """Half a step of `dtype` at the value, and half its smallest number."""
    f = torch.finfo(dtype)
    return value.abs() * (f.eps / 2) + f.smallest_normal * f.eps / 2


def assert_within(got, want, tol, what=""):
    """Equal infinities and NaN in the same places, everything else within the bound; past the range of got's type is infinite."""
    most = torch.finfo(got.dtype).max   # of fp16: 65504, so that a gradient of 1 / T = 1e6 is infinite
    got, want = got.detach().double(), want.double()
    want = torch.where(want.abs() > most, want.sign() * np.inf, want)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    special = torch.isnan(want) | torch.isinf(want)
    assert torch.equal(torch.where(torch.isinf(want), got, want)[~torch.isnan(want)], want[~torch.isnan(want)]), what
    off = torch.where(special, torch.zeros_like(want), (got - want).abs())
    tol = torch.where(special, torch.ones_like(want), tol.double().expand_as(want) if torch.is_tensor(tol) else torch.full_like(want, tol))
    worst = (off - tol).max().item() if off.numel() else -1.0
    assert worst <= 0, (what, worst, off.max().item())


def make_logits(rows, cats, dtype, seed, spread=3.0, device="cuda"):
    gen = torch.Generator(device="cpu")
    gen.manual_seed(seed)
    x = spread * torch.randn(rows, cats, generator=gen) + 5.0 * torch.randn(rows, 1, generator=gen)
    return x.to(dtype).to(device)
