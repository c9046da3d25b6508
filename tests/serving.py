"""Plain float64 implementations of the serving operators (8-bit caches,
windows with first tokens, block moves) and their error bounds, for the tests."""

import math

import torch

F8 = torch.float8_e4m3fn
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11}


# ------------------------------------------------------------- 8-bit blocks --
def round_e4m3(x):
    """float64 -> the nearest e4m3 value, ties to even, as float64; beyond 448 to 448, NaN stays."""
    _, e = torch.frexp(x)
    step = torch.exp2((e - 4).clamp(min=-9).double())
    y = torch.where(x == 0, x, torch.round(x / step) * step)
    y = torch.where(x.abs() == math.inf, torch.sign(x) * 448.0, y)
    return y.clamp(-448.0, 448.0)


def fit_scale(x):
    """2^e, the smallest e >= -126 with max |x| <= 448 * 2^e over the finite x."""
    top = torch.where(torch.isfinite(x), x.abs(), 0.0).max().item() if x.numel() else 0.0
    e = -126
    if top > 0:
        e = max(-126, math.frexp(top)[1] - 9)
        while 448.0 * 2.0 ** e < top:
            e += 1
        while e > -126 and 448.0 * 2.0 ** (e - 1) >= top:
            e -= 1
    return 2.0 ** e


def append(codes, scale, rows, lens, table, page):
    """rows[i] [n_i, heads, dim] float64 appended at lens[i]: codes (float64, [blocks, heads, page, dim]) and scale
    (float64 [blocks, heads]) change in place."""
    for i, n in enumerate(lens):
        if n < 0:
            continue
        r = rows[i]
        for p in range(n // page, -(-(n + r.shape[0]) // page)):
            a, z = max(n, p * page), min(n + r.shape[0], (p + 1) * page)
            if a >= z or p >= len(table[i]) or not 0 <= table[i][p] < codes.shape[0]:
                continue
            b = table[i][p]
            for h in range(codes.shape[1]):
                x = r[a - n:z - n, h]
                old = 0.0 if a == p * page else scale[b, h].item()
                now = max(old, fit_scale(x))
                if a != p * page and now != old:
                    codes[b, h] = round_e4m3(codes[b, h] * (old / now))
                scale[b, h] = now
                codes[b, h, a - p * page:z - p * page] = round_e4m3(x / now)


# ---------------------------------------------------------------- attention --
def seen_decode(L, left, sinks):
    """Positions a query at L - 1 sees."""
    return [t for t in range(L) if left < 0 or t >= L - 1 - left or t < sinks]


def attention(q, k, v, seen, scale):
    """q [rows, d], k/v [keys, d], seen [rows, keys] (float64): out, lse, and the magnitudes the error bounds need:
    sum p |v| and the largest scale * sum |q| |k| over the seen keys."""
    w = (q @ k.T * scale).masked_fill(~seen, -math.inf)
    m = w.amax(-1, keepdim=True) if k.shape[0] else torch.full((q.shape[0], 1), -math.inf, dtype=torch.float64)
    m = torch.where(m == -math.inf, 0.0, m)
    p = torch.exp(w - m)
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    lse = (m + torch.log(total)).squeeze(-1)
    size = (q.abs() @ k.abs().T * abs(scale)).masked_fill(~seen, 0.0)
    top = size.amax(-1) if k.shape[0] else torch.zeros(q.shape[0], dtype=torch.float64)
    return p @ v, lse, p @ v.abs(), top


def bound(ref, spread, top, d, keys, out_dtype, weight_step, query_step=0.0):
    """How far a kernel's output may be from ref: its own rounding, the rounding of the weights (weight_step), the
    scores' error (d products summed in fp32, the query's rounding), the exponentials (2^-21) and the sums over keys
    in fp32, each relative to sum p |v|."""
    score = top * ((d + 8) * 2.0 ** -23 + query_step)
    inner = weight_step + 2 * torch.expm1(score) + 2.0 ** -20 + (keys / 16 + 40) * 2.0 ** -23
    return HALF_STEP[out_dtype] * ref.abs() + inner[:, None] * spread + 1e-30


# ------------------------------------------------------------------- layout --
def unpack(cache, k_side, kind):
    """[blocks, heads, page, dim] rows of a float cache's blocks."""
    n, h, page, d = cache.shape
    if kind == "8bit" or not k_side:
        return cache
    if cache.dtype == torch.bfloat16:
        return cache.reshape(n, h, d // 2, page, 2).transpose(2, 3).reshape(n, h, page, d)
    return cache.reshape(n, h, d, page).transpose(2, 3)


def pack(rows, k_side, kind):
    """The inverse of unpack."""
    n, h, page, d = rows.shape
    if kind == "8bit" or not k_side:
        return rows.contiguous()
    if rows.dtype == torch.bfloat16:
        return rows.reshape(n, h, page, d // 2, 2).transpose(2, 3).reshape(n, h, page, d).contiguous()
    return rows.transpose(2, 3).reshape(n, h, page, d).contiguous()


class Paged:
    """Random paged caches: every sequence has its blocks in a shuffled order, and what no sequence uses -- slots past
    a length, blocks of nobody, pages behind a window -- holds NaN; freed table entries hold garbage."""

    def __init__(self, kind, lens, kv_heads, d, page, dtype, seed=0, left=-1, sinks=0, room=0, device="cuda", own=None,
                 even=False):
        # own: whether an 8-bit cache's scales are no powers of two (a user's own); by the seed when None.
        # even: its values are near N(0, 1), so that scores differ by a few units and many keys carry weight.
        own = bool(seed % 2) if own is None else own
        g = torch.Generator().manual_seed(seed)
        self.kind, self.lens, self.page, self.left, self.sinks = kind, list(lens), page, left, sinks
        ends = [-(-(n + room) // page) if n >= 0 else 0 for n in lens]
        width = max(1, max(ends, default=1))
        total = sum(ends) + 2
        order = torch.randperm(total, generator=g).tolist()
        table, at = [], 0
        for e in ends:
            table.append(order[at:at + e] + [order[-1]] * (width - e))
            at += e
        self.table = table
        rows = [torch.randn(total, kv_heads, page, d, generator=g, dtype=torch.float64) for _ in range(2)]
        self.scale = [None, None]
        if kind == "8bit":
            dt = F8
            for x in range(2):
                s = torch.exp2(torch.randint(*((-1, 2) if even else (-9, 3)), (total, kv_heads), generator=g).double())
                rows[x] = round_e4m3(rows[x] * 100)
                if even:
                    s = s * (1.28 if own else 1) / 128
                else:
                    s = s / 100 if own else s
                self.scale[x] = s
                self.scale[x] = self.scale[x].float().double()
        else:
            dt = dtype
            rows = [r.to(dtype).double() for r in rows]
        # what a sequence may be asked for, kept as float64
        self.rows = [r.clone() for r in rows]
        keep = torch.zeros(total, page, dtype=torch.bool)
        for i, n in enumerate(lens):
            for p in range(ends[i]):
                pos = torch.arange(p * page, (p + 1) * page)
                keep[table[i][p]] = pos < n
        for r in rows:
            r.masked_fill_(~keep[:, None, :, None], math.nan)
        self.k_cache, self.v_cache = (pack(r.float().to(dt) if kind == "8bit" else r.to(dt), x == 0, kind).to(device)
                                      for x, r in enumerate(rows))
        self.k_scale, self.v_scale = (None if s is None else s.float().to(device) for s in self.scale)
        if left >= 0:
            for i, n in enumerate(lens):
                for p in range(ends[i]):
                    if p * page >= sinks and (p + 1) * page <= n + room - 1 - left:
                        table[i][p] = -1 if i % 2 else 0x7fffffff
        self.bt = torch.tensor(table, dtype=torch.int32).reshape(len(lens), width).to(device)
        self.L = torch.tensor(self.lens, dtype=torch.int32, device=device)

    def opts(self):
        return {} if self.kind != "8bit" else dict(k_descale=self.k_scale, v_descale=self.v_scale)

    def keys(self, i, h, positions, side):
        if not len(positions):
            return torch.zeros(0, self.rows[0].shape[-1], dtype=torch.float64)
        b = torch.tensor([self.table[i][t // self.page] for t in positions])
        o = torch.tensor([t % self.page for t in positions])
        r = self.rows[side][b, h, o]
        return r if self.scale[side] is None else r * self.scale[side][b, h][:, None]


def check_decode(out, lse, q, pc, heads, scale=None, lens=None):
    """Checks out [B, 1, H, d] (and lse [B, H, 1]) against the definition, with the derived bound."""
    kv = pc.rows[0].shape[1]
    d = q.shape[-1]
    scale = d ** -0.5 if scale is None else scale
    group = heads // kv
    fp32 = q.dtype == torch.float32
    # 8-bit caches under bf16 queries: a weight is one f16 value, half a step 2^-11. The largest weight * scale is 2^6 or
    # more, so below f16's normal range the half step 2^-25 is 2^-31 of it: keys * 2^-31 * max |v| in all. Under fp32
    # queries it is two f16 values: 2^-11 squared. bf16 caches: two bf16 values, 2^-8 squared.
    eight = pc.kind == "8bit"
    weight = {"8bit": 2.0 ** -22 if fp32 else 2.0 ** -11, "bf16": 2.0 ** -16, "fp32": 0.0}[pc.kind]
    query = 2.0 ** -22 if pc.kind == "8bit" else 0.0
    got = out.double().cpu()
    for i, n in enumerate(pc.lens if lens is None else lens):
        pos = seen_decode(max(n, 0), pc.left, pc.sinks)
        for h in range(kv):
            k, v = (pc.keys(i, h, pos, x) for x in (0, 1))
            qq = q[i, 0, h * group:(h + 1) * group].double().cpu()
            ref, z, spread, top = attention(qq, k, v, torch.ones(group, len(pos), dtype=torch.bool), scale)
            tol = bound(ref, spread, top, d, len(pos), q.dtype, weight, query)
            if eight and len(pos):
                tol = tol + len(pos) * 2.0 ** -31 * v.abs().amax(0)
            err = (got[i, 0, h * group:(h + 1) * group] - ref).abs()
            assert (err <= tol).all(), (i, h, err.max().item(), (err / tol).max().item())
            if lse is not None:
                zz = lse[i, h * group:(h + 1) * group, 0].double().cpu()
                if not pos:
                    assert torch.isneginf(zz).all()
                else:
                    slack = top * ((d + 8) * 2.0 ** -23 + query) + 2.0 ** -19 + 2.0 ** -22 * z.abs() \
                        + (len(pos) / 16) * 2.0 ** -23
                    assert ((zz - z).abs() <= slack).all(), (i, h, (zz - z).abs().max().item())
