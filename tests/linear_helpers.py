"""The linear-attention operators' definitions in float64, row after row, with bounds on what float32 may be
off, and inputs for their tests."""
import numpy as np
import torch

from bitgpu_amd import engine as E

U = 2.0 ** -24  # half a step of float32


def cuda(x):
    return None if x is None else torch.from_numpy(np.ascontiguousarray(x, np.float32)).cuda()


def unit(x):
    return x / np.sqrt((x * x).sum(-1, keepdims=True) + 1e-6)


def silu(x):
    return x / (1 + np.exp(-x))


class Case:
    """Inputs of one call: ragged rows of several sequences with slots and sources."""

    def __init__(self, rows, Hk=2, Hv=4, dk=128, dv=128, rule="delta", gate=False, norm=False, const_g=False, seed=0, slots=None,
                 sources=None, spare=2, corr=0.3):
        rng = np.random.default_rng(seed)
        self.rows, self.Hk, self.Hv, self.dk, self.dv, self.rule = list(rows), Hk, Hv, dk, dv, rule
        T, B = sum(rows), len(rows)
        self.T, self.n_slots = T, B + spare
        self.slots = list(rng.permutation(self.n_slots)[:B]) if slots is None else slots
        self.slots = [int(s) for s in self.slots]
        self.sources = sources
        n = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
        # keys of a sequence share a direction, as those behind a SiLU do
        self.k = unit(n(T, Hk, dk) + corr * np.sqrt(dk) * unit(n(1, Hk, dk))).astype(np.float32)
        self.q = unit(n(T, Hk, dk)).astype(np.float32)
        self.v = n(T, Hv, dv)
        rate = np.exp(rng.uniform(-6, 0.5, Hv)).astype(np.float32)
        self.g = -rate if const_g else (-rate * np.exp(0.5 * n(T, Hv))).astype(np.float32)
        self.beta = (1 / (1 + np.exp(-n(T, Hv)))).astype(np.float32) if rule == "delta" else None
        self.norm = (1 + 0.1 * n(dv)) if norm or gate else None
        self.z = n(T, Hv, dv) if gate else None
        self.state = 0.3 * n(1, self.n_slots, Hv, dv, dk)
        self.eps = 1e-6

    def cache(self, **more):
        return E.LinearStateCache(1, self.Hk, self.Hv, self.dk, self.dv, n_slots=self.n_slots, conv_width=0,
                                  state=cuda(self.state), **more)

    def run(self, cache=None, batch=None, out=None):
        """(out, state) of the framework's call."""
        cache = cache or self.cache()
        if batch is None:
            batch = E.LinearBatch(cache, max(1, len(self.rows)), max(1, self.T))
            batch.set(self.rows, self.slots, self.sources)
        out = E.linear_attention(cache, 0, batch, cuda(self.q), cuda(self.k), cuda(self.v), cuda(self.g), cuda(self.beta),
                                 gate=cuda(self.z), norm=cuda(self.norm), eps=self.eps, out=out)
        torch.cuda.synchronize()
        return out.cpu().numpy(), cache.state.cpu().numpy()

    def check(self, out, state):
        want, bound, S, S_bound = self.reference()
        err = np.abs(out - want)
        assert np.all(err <= bound), f"out: {np.nanmax(err / bound):.3g} of the bound at {np.unravel_index(np.nanargmax(err / bound), err.shape)}"
        err = np.sqrt(np.square(state - S).sum(-1))
        assert np.all(err <= S_bound), f"state: {np.nanmax(err / np.maximum(S_bound, 1e-300)):.3g} of the bound"

    def reference(self):
        """out, its bound, the states, and the bound of a state row's error (2-norm).

        The bound follows the recurrence in 2-norms over the key dims, for each value dim. A row's fade and
        write map an error e of the state row to at most |e| (fade <= 1; 1 - beta k k^T has norm <= 1 for
        |k| <= 1 and 0 <= beta <= 1), and round by at most N U of the sizes that enter: |S| for the fade, the
        sum and the dot product with the key (|k| <= 1), |v| for the correction. N = dk / 8 + 8 covers a dot
        product in eight lanes, the decay's exp (2 ulp) and the update's own roundings; the same N covers
        products of operands held to 2^-22 each (2^-20.4 together, N U >= 2^-20) summed in any order up to
        that depth. A chunk's rows are corrected through (I + A)^-1 instead: errors of its right-hand side and
        its own roundings grow by at most its norm, taken as the largest row sum of |.| over the case. The
        output reads the state with |q| <= 1. The norm behind it divides by its rms: twice the relative
        change, plus 16 roundings; SiLU's argument is exact and its value within 8 U."""
        T, Hv, rep, dk, dv = self.T, self.Hv, self.Hv // self.Hk, self.dk, self.dv
        N = dk / 8 + 8
        f64 = lambda x: None if x is None else np.asarray(x, np.float64)  # noqa: E731
        q, k, v, g, beta = f64(self.q), f64(self.k), f64(self.v), f64(self.g), f64(self.beta)
        g = np.broadcast_to(g, (T, Hv))
        out, bound = np.zeros((T, Hv, dv)), np.zeros((T, Hv, dv))
        states, errors = f64(self.state).copy(), np.zeros((1, self.n_slots, Hv, dv))
        start = f64(self.state)
        at = 0
        sources = self.slots if self.sources is None else self.sources
        grow = self.growth() if self.rule == "delta" else 1.0
        for r, slot, src in zip(self.rows, self.slots, sources):
            if r == 0:
                continue
            S = start[0, src].copy() if src >= 0 else np.zeros((Hv, dv, dk))
            e = np.zeros((Hv, dv))
            for t in range(at, at + r):
                kk, qq = np.repeat(k[t], rep, 0), np.repeat(q[t], rep, 0)
                a = np.exp(g[t])[:, None]
                size = np.sqrt(np.square(S).sum(-1))
                S = S * a[..., None]
                d = v[t]
                if beta is not None:
                    d = beta[t][:, None] * (v[t] - np.einsum("hvk,hk->hv", S, kk))
                S = S + d[..., None] * kk[:, None]
                after = np.sqrt(np.square(S).sum(-1))
                e = a * e + N * U * grow * (a * size + after + np.abs(v[t]))
                out[t] = np.einsum("hvk,hk->hv", S, qq) / np.sqrt(dk)
                bound[t] = (e + N * U * grow * (size + after + np.abs(v[t]))) / np.sqrt(dk)
            states[0, slot], errors[0, slot] = S, e
            at += r
        if self.norm is not None:
            rms = np.sqrt(np.square(out).mean(-1, keepdims=True) + self.eps)
            off = np.sqrt(np.square(bound).mean(-1, keepdims=True)) / rms
            w = f64(self.norm) * (silu(f64(self.z)) if self.z is not None else 1)
            out, bound = out / rms * w, np.abs(w) * (bound / rms + np.abs(out) / rms * (2 * off + 24 * U))
        return out, bound + 1e-30, states, errors + 1e-30

    def growth(self):
        """The largest absolute row sum of (I + A)^-1 over the sequences' chunks of 64 rows, at least 1."""
        most, at, rep = 1.0, 0, self.Hv // self.Hk
        g = np.broadcast_to(np.asarray(self.g, np.float64), (self.T, self.Hv))
        for r in self.rows:
            for c in range(at, at + r, 64):
                n = min(64, at + r - c)
                s = np.cumsum(g[c:c + n], 0)
                for h in range(self.Hv):
                    kk = self.k[c:c + n, h // rep].astype(np.float64)
                    A = np.tril(self.beta[c:c + n, h, None] * (kk @ kk.T) * np.exp(np.minimum(s[:, None, h] - s[None, :, h], 0)), -1)
                    most = max(most, np.abs(np.linalg.inv(np.eye(n) + A)).sum(-1).max())
            at += r
        return most
