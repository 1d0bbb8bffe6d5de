"""Plain restatements in 64 bits, on the CPU, of the 8-bit cache and of the token log probabilities: loops over sequences, pages
and heads, written from the definitions at tvae_kv8_* / tvae_token_logp in include/tvae_kernels.h."""
import math

import torch

E_MIN, E_MAX = 27, 246


def code_values():
    "float64 value of each of the 256 codes: 1 sign, 4 exponent (bias 7), 3 mantissa bits, 0x7F / 0xFF NaN"
    out = []
    for b in range(256):
        e, m = (b >> 3) & 15, b & 7
        v = math.nan if (b & 127) == 127 else m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        out.append(-v if b & 128 else v)
    return torch.tensor(out, dtype=torch.float64)


VALUES = code_values()
_POS = VALUES[:127]                                    # 0 .. 448, ascending


def encode(y):
    "float64 values -> codes: nearest, halves to the even code, clamped to +-448, non-finite -> 0x7F"
    a = y.abs().clamp(max=448.0)
    hi = torch.searchsorted(_POS, a.contiguous()).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    dl, dh = a - _POS[lo], _POS[hi] - a
    pick = torch.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    code = torch.where(torch.signbit(y), pick + 128, pick)
    return torch.where(torch.isfinite(y), code, torch.full_like(code, 127)).to(torch.uint8)


def need_exp(x):
    "stored exponent for the values x"
    x = x[torch.isfinite(x)].abs()
    top = float(x.max()) if x.numel() else 0.0
    if top == 0.0:
        return E_MIN
    m, e = math.frexp(top)                             # top = m 2^e, 0.5 <= m < 1; 448 = 0.875 * 2^9
    return min(E_MAX, max(E_MIN, e - 9 + (1 if m > 0.875 else 0) + 127))


class Cache:
    "the four arrays on the CPU"

    def __init__(self, n_pages, h, dk, page):
        self.k, self.v = (torch.zeros((n_pages, h, page, dk), dtype=torch.uint8) for _ in range(2))
        self.ke, self.ve = (torch.full((n_pages, h), 127, dtype=torch.uint8) for _ in range(2))
        self.n_pages, self.h, self.page, self.dk = n_pages, h, page, dk

    def page_of(self, table, per, b, slot):
        p = b * per + slot if table is None else int(table[b, slot])
        return p if 0 <= p < self.n_pages else None

    def store(self, k, v, start, count, table, per):
        n, T = k.shape[:2]
        for codes, exps, x in ((self.k, self.ke, k), (self.v, self.ve, v)):
            for b in range(n):
                if start[b] < 0:
                    continue
                end = min(start[b] + max(0, min(T, count[b])), per * self.page)
                pos = start[b]
                while pos < end:
                    slot, at = divmod(pos, self.page)
                    to = min(self.page, at + end - pos)
                    p = self.page_of(table, per, b, slot)
                    if p is not None:
                        rows = x[b, pos - start[b]:pos - start[b] + to - at].double()            # (rows, h, dk)
                        for i in range(self.h):
                            e = need_exp(rows[:, i])
                            if at:
                                old = min(int(exps[p, i]), E_MAX)
                                e = max(e, old)
                                if e > old:
                                    codes[p, i, :at] = encode(VALUES[codes[p, i, :at].long()] * 2.0 ** (old - e))
                            codes[p, i, at:to] = encode(rows[:, i] * 2.0 ** (127 - e))
                            exps[p, i] = e
                    pos += to - at

    def load(self, T, start, count, table, per, n):
        out = []
        for codes, exps in ((self.k, self.ke), (self.v, self.ve)):
            o = torch.zeros((n, T, self.h, self.dk), dtype=torch.float64)
            for b in range(n):
                for t in range(min(T, count[b])):
                    pos = start[b] + t
                    if 0 <= pos < per * self.page:
                        p = self.page_of(table, per, b, pos // self.page)
                        if p is not None:
                            o[b, t] = VALUES[codes[p, :, pos % self.page].long()] * torch.exp2(exps[p].double() - 127)[:, None]
            out.append(o)
        return out

    def attend(self, q, lens, table, per, causal=True, mask=None, scale=None):
        """(o, weights' sum of |v|, largest sum of |q k| scale): the second and third are what a rounding error of the weights
        and of the scores is multiplied by."""
        n, Lq, hq, dk = q.shape
        G = hq // self.h
        scale = 1 / math.sqrt(dk) if scale is None else scale
        o, wv, qk = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape[:3], dtype=torch.float64)
        for b in range(n):
            L = max(0, min(int(lens[b]), per * self.page))
            live = torch.zeros(L, dtype=torch.bool)
            kk, vv = torch.zeros((L, self.h, dk), dtype=torch.float64), torch.zeros((L, self.h, dk), dtype=torch.float64)
            for a in range(0, L, self.page):
                p = self.page_of(table, per, b, a // self.page)
                if p is None:
                    continue
                z = min(L, a + self.page)
                live[a:z] = True
                kk[a:z] = (VALUES[self.k[p, :, :z - a].long()] * torch.exp2(self.ke[p].double() - 127)[:, None, None]).transpose(0, 1)
                vv[a:z] = (VALUES[self.v[p, :, :z - a].long()] * torch.exp2(self.ve[p].double() - 127)[:, None, None]).transpose(0, 1)
            if mask is not None:
                w = min(L, mask.shape[1])
                live[:w] &= mask[b, :w].bool()
                live[w:] = False
            for i in range(Lq):
                see = live.clone()
                if causal:
                    see[max(0, L - (Lq - 1 - i)):] = False
                if not bool(see.any()):
                    continue
                for g in range(hq):
                    qi, ki, vi = q[b, i, g].double(), kk[see, g // G], vv[see, g // G]
                    w = torch.softmax(ki @ qi * scale, 0)
                    o[b, i, g], wv[b, i, g] = w @ vi, w @ vi.abs()
                    qk[b, i, g] = (ki.abs() @ qi.abs()).max() * abs(scale)
        return o, wv, qk


def attend_bound(o, wv, qk, dk, keys, dtype):
    """How far an fp32 kernel may be from o.  A score is a sum of dk products: off by (dk + 8) 2^-24 of sum |q k| scale, at most qk;
    that moves every weight, and their sum, by as much relative.  exp2 and its argument: 2^-21.  The sums over the keys:
    (keys + 64) 2^-24.  In 16-bit types the weights may be rounded to that type on their way into the second product: half a
    step of it (eps / 2).  At last the result's own rounding, half a step (a denormal's step below the normal range)."""
    half = torch.finfo(dtype).eps / 2
    rel = 2 * (dk + 8) * 2.0 ** -24 * qk + 2.0 ** -21 + (keys + 64) * 2.0 ** -24 + (half if dtype != torch.float32 else 0.0)
    return rel[..., None] * wv + half * o.abs() + torch.finfo(dtype).smallest_normal


def _shifted(logits):
    "the logits in float64 less their row's maximum, which changes no probability: 1e38 + ln V is 1e38 in 64 bits too"
    x = logits.double()
    top = x.nan_to_num(nan=-math.inf, posinf=math.inf, neginf=-math.inf).amax(1, keepdim=True)
    return x - torch.where(torch.isfinite(top), top, torch.zeros_like(top))


def score(logits, tokens, top):
    "(logp, entropy, top_logp, top_ids) in float64"
    x = _shifted(logits)
    rows, V = x.shape
    lse = torch.logsumexp(x, 1)
    lp = x - lse[:, None]
    none = torch.isneginf(lse)
    lp[none] = -math.inf
    p = lp.exp()
    ent = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(1)
    ent[torch.isnan(lse) | torch.isposinf(lse)] = math.nan
    lp[torch.isposinf(lse)] = math.nan
    logp = torch.zeros(rows, dtype=torch.float64)
    if tokens is not None:
        ok = (tokens >= 0) & (tokens < V)
        logp[ok] = lp[ok, tokens[ok]]
    ids = torch.zeros((rows, top), dtype=torch.int64)
    x = logits.double()
    for r in range(rows):
        order = sorted(range(V), key=lambda c: (0 if math.isnan(x[r, c]) else 1, 0.0 if math.isnan(x[r, c]) else -float(x[r, c]), c))
        ids[r] = torch.tensor(order[:top], dtype=torch.int64)
    return logp, ent, lp.gather(1, ids), ids


def score_grad(logits, tokens, ids, g_logp, g_ent, g_top):
    "gradient of sum(g_logp logp) + sum(g_ent H) + sum(g_top top_logp), from the formula"
    x = _shifted(logits)
    rows, V = x.shape
    lse = torch.logsumexp(x, 1)
    lp = x - lse[:, None]
    p = lp.exp()
    none = torch.isneginf(lse)
    H = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(1)
    lpz = torch.where(p > 0, lp, torch.zeros_like(lp))
    ok = torch.zeros(rows, dtype=torch.bool) if tokens is None else (tokens >= 0) & (tokens < V)
    gl = torch.where(ok, g_logp.double(), torch.zeros(rows, dtype=torch.float64)) if g_logp is not None else torch.zeros(rows, dtype=torch.float64)
    ge = g_ent.double() if g_ent is not None else torch.zeros(rows, dtype=torch.float64)
    gt = g_top.double() if g_top is not None else torch.zeros((rows, 0), dtype=torch.float64)
    dx = -p * ((gl + gt.sum(1))[:, None] + ge[:, None] * (lpz + H[:, None]))
    for r in range(rows):
        if ok[r]:
            dx[r, int(tokens[r])] += gl[r]
        for t in range(gt.shape[1]):
            dx[r, int(ids[r, t])] += gt[r, t]
    dx[torch.isneginf(x)] = 0.0
    dx[none] = 0.0
    return dx
