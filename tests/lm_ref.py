"""The language model in float64 from a pack's weights, with an optional window and sinks: every row of keys and values is kept and a mask
says what a row sees, so nothing of a paged cache's bookkeeping is repeated here."""
import math

import numpy as np


class Lm:
    def __init__(self, spec, weights, window=0, sinks=0):
        self.s, self.w, self.window, self.sinks = spec, {k: np.asarray(v, np.float64) for k, v in weights.items() if k.startswith("lm.")}, window, sinks
        self.keys = [np.zeros((0, spec.d_model)) for _ in range(spec.lm_layers)]
        self.values = [np.zeros((0, spec.d_model)) for _ in range(spec.lm_layers)]
        self.length = 0

    def _norm(self, x, g, b):
        x = x - x.mean(-1, keepdims=True)
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + self.s.lm_ln_eps) * self.w[g] + self.w[b]

    def _turn(self, x, pos):
        half = self.s.d_model // self.s.lm_heads // 2
        angle = pos[:, None] * float(self.s.lm_max_period) ** (-np.arange(half) / half)
        c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
        y = x.reshape(len(x), self.s.lm_heads, half, 2)
        return np.stack([y[..., 0] * c - y[..., 1] * s, y[..., 0] * s + y[..., 1] * c], -1).reshape(len(x), -1)

    def rows(self, x):
        """New rows x [n][d_model]; returns (conditioning [d_model], EOS logit) of the last."""
        s, d, dh = self.s, self.s.d_model, self.s.d_model // self.s.lm_heads
        x = np.array(x, np.float64)
        pos = self.length + np.arange(len(x))
        self.length += len(x)
        j = np.arange(self.length)[None]
        see = j <= pos[:, None]
        if self.window:
            see &= (j > pos[:, None] - self.window) | (j < self.sinks)
        for i in range(s.lm_layers):
            p = f"lm.l{i}."
            q, k, v = np.split(self._norm(x, p + "ln1.g", p + "ln1.b") @ self.w[p + "qkv.w"].T, 3, -1)
            self.keys[i] = np.concatenate([self.keys[i], self._turn(k, pos)])
            self.values[i] = np.concatenate([self.values[i], v])
            q, out = self._turn(q, pos), np.empty_like(x)
            for h in range(0, d, dh):
                a = q[:, h:h + dh] @ self.keys[i][:, h:h + dh].T / math.sqrt(dh)
                a = np.exp(np.where(see, a, -np.inf) - np.where(see, a, -np.inf).max(-1, keepdims=True))
                out[:, h:h + dh] = a @ self.values[i][:, h:h + dh] / a.sum(-1, keepdims=True)
            x = x + out @ self.w[p + "out.w"].T
            f = self._norm(x, p + "ln2.g", p + "ln2.b") @ self.w[p + "ff1.w"].T
            f = 0.5 * f * (1 + np.vectorize(math.erf)(f / math.sqrt(2)))
            x = x + f @ self.w[p + "ff2.w"].T
        last = self._norm(x[-1], "lm.out_norm.g", "lm.out_norm.b")
        return last, float(last @ self.w["lm.eos.w"].reshape(-1) + self.w["lm.eos.b"].reshape(-1)[0])

    def latent(self, z):
        """One latent frame (NaN: the start of the sequence)."""
        z = np.where(np.isnan(z), self.w["lm.bos_emb"], z)
        return self.rows((self.w["lm.in_proj.w"] @ z)[None])
