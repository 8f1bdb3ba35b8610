"""The sequence operators as a user calls them, with plain forms of the same arithmetic beside them.

Three operators: the gated linear recurrence (forward, backward, one-event step), attention of a batch of queries that share
a long prefix, and dropout whose keep decisions come from a counter-based generator.  ``own`` false: elementary torch
operations in 32 bits, rounded once at the end; ``own`` true: the framework's entry points.
"""
import math

import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
WORD = (1 << 64) - 1
GOLDEN, MIX1, MIX2 = 0x9E3779B97F4A7C15, 0xBF58476D1CE4E5B9, 0x94D049BB133111EB


# ------------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # 128 sequences of 100 events, 32 units (the Amazon configuration's batch): the small training step of one layer
        dict(name="scan_train_amazon", op="scan", train=True, B=128, T=100, C=32, dtype="fp32", period=2, pad=True, h0=False),
        # the XLong configuration's first layer: 500 sequences, 1024 steps, 64 units, every second state handed on
        dict(name="scan_train_xlong", op="scan", train=True, B=500, T=1024, C=64, dtype="fp32", period=2, pad=False, h0=False),
        # a wide bf16 layer over long sequences, every state handed on, starting from carried states
        dict(name="scan_train_wide_bf16", op="scan", train=True, B=16, T=4096, C=1024, dtype="bf16", period=1, pad=False, h0=True),
        # odd sizes in fp16 with front padding, a sequence without any event among them
        dict(name="scan_train_odd_fp16", op="scan", train=True, B=37, T=517, C=100, dtype="fp16", period=1, pad=True, h0=True),
        # one user's whole life in one call (state store rebuilt from the log): few rows, a long axis
        dict(name="scan_infer_one_long", op="scan", train=False, B=1, T=65536, C=256, dtype="bf16", period=1, pad=False, h0=True),
        # one candidate event scored against one stored user: latency
        dict(name="step_one", op="step", B=1, C=64, users=1000, dtype="fp32"),
        # a ranking request's batch of candidate events over a store of users
        dict(name="step_batch", op="step", B=4096, C=128, users=65536, dtype="bf16"),
        # the head's hidden layer of one batch: latency
        dict(name="dropout_head", op="dropout", N=128, C=200, dtype="fp32", keep=0.5, residual=False),
        # activations of a long bf16 batch, added to the residual stream
        dict(name="dropout_wide_bf16", op="dropout", N=65536, C=1024, dtype="bf16", keep=0.9, residual=True),
        # a few candidates against one user's thousand events, the framework's own type
        dict(name="attn_few_fp32", op="attn", B=8, Lq=1, Hq=1, Hkv=1, D=64, P=1000, S=0, dtype="fp32", lse=True),
        # 200 candidates, grouped heads, each with a short session of its own behind a long shared history
        dict(name="attn_rank_bf16", op="attn", B=200, Lq=1, Hq=8, Hkv=2, D=64, P=4096, S=32, dtype="bf16", lse=False),
        # the largest: 512 rows, 16 heads of 128, a prefix of 32768
        dict(name="attn_large_bf16", op="attn", B=512, Lq=1, Hq=16, Hkv=4, D=128, P=32768, S=64, dtype="bf16", lse=False),
    ]


def _between(rng, lo, hi):
    """A whole number in [lo, hi], evenly over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["scan", "scan", "step", "dropout", "attn", "attn"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op == "scan":
        period = rng.choice([1, 1, 2, 3, 5])
        while True:
            B, C = _between(rng, 1, 500), _between(rng, 1, 1024)
            T = period * _between(rng, 1, 65536 // period)
            if B * T * C <= 1 << 25:
                return dict(op="scan", train=rng.random() < 0.7, B=B, T=T, C=C, dtype=dtype, period=period, pad=rng.random() < 0.5,
                            h0=rng.random() < 0.5)
    if op == "step":
        B = _between(rng, 1, 4096)
        return dict(op="step", B=B, C=_between(rng, 1, 512), users=B + _between(rng, 1, 60000), dtype=dtype)
    if op == "dropout":
        return dict(op="dropout", N=_between(rng, 1, 32768), C=_between(rng, 1, 1024), dtype=dtype, keep=rng.choice([0.5, 0.8, 0.9, 0.95]),
                    residual=rng.random() < 0.5)
    while True:
        Lq = 1 if rng.random() < 0.7 else _between(rng, 2, 48)
        c = dict(op="attn", B=_between(rng, 1, 512), Lq=Lq, Hkv=rng.choice([1, 2, 3, 4, 8]), D=rng.choice([32, 40, 64, 64, 72, 96, 128, 128]),
                 P=_between(rng, 1, 32768), S=rng.choice([0, Lq, Lq + _between(rng, 1, 300)]), dtype=dtype, lse=rng.random() < 0.3)
        c["Hq"] = c["Hkv"] * rng.choice([1, 2, 4, 5, 8])
        if work(c)["flops"] <= 3e10 and c["B"] * c["Hkv"] * c["S"] * c["D"] <= 1 << 26:
            return c


def work(c):
    s = SIZE[c["dtype"]]
    if c["op"] == "scan":
        n, y = c["B"] * c["T"] * c["C"], c["B"] * (c["T"] // c["period"]) * c["C"]
        if c["train"]:
            return {"bytes": (4 * n + 2 * y) * s, "flops": 24 * n}
        return {"bytes": (2 * n + y) * s, "flops": 8 * n}
    if c["op"] == "step":
        return {"bytes": c["B"] * c["C"] * (3 * s + 4), "flops": 8 * c["B"] * c["C"]}
    if c["op"] == "dropout":
        return {"bytes": c["N"] * c["C"] * s * (5 if c["residual"] else 4), "flops": 3 * c["N"] * c["C"]}
    rows, own_keys = c["B"] * c["Lq"] * c["Hq"], c["S"] / 2
    return {"bytes": (2 * c["P"] * c["Hkv"] + c["B"] * c["S"] * c["Hkv"] + 2 * rows) * c["D"] * s,
            "flops": 4 * rows * (c["P"] + own_keys) * c["D"]}


# ----------------------------------------------------------------------------------------------------------------- inputs
def prepare(c, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    t = TYPES[c["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    st = dict(c)
    if c["op"] == "scan":
        B, T, C, p = c["B"], c["T"], c["C"], c["period"]
        # gates and candidates come out of one projection side by side; the gates carry the GRU's bias of 1
        proj = torch.empty(B, T, 2 * C, device=dev, dtype=t)
        proj[..., :C] = (1.0 + 1.5 * normal(B, T, C)).to(t)
        proj[..., C:] = torch.tanh(normal(B, T, C)).to(t)
        st["proj"] = proj
        st["begin"] = None
        if c["pad"]:
            begin = (torch.rand(B, device=dev, generator=g) * T).to(torch.int32)
            begin[-1] = 0                                  # no padding
            if B > 1:
                begin[0] = T                               # nothing but padding
            st["begin"] = begin
        st["start"] = 0.5 * normal(B, C) if c["h0"] else None
        if c["train"]:
            st["d_y"] = normal(B, T // p, C).to(t)
            st["d_h_last"] = normal(B, C)
    elif c["op"] == "step":
        st["z"] = (1.0 + 1.5 * normal(c["B"], c["C"])).to(t)
        st["v"] = torch.tanh(normal(c["B"], c["C"])).to(t)
        st["store"] = 0.5 * normal(c["users"], c["C"])
        st["user"] = torch.randint(0, c["users"], (c["B"],), device=dev, generator=g, dtype=torch.int32)
    elif c["op"] == "dropout":
        st["x"] = normal(c["N"], c["C"]).to(t)
        st["res"] = normal(c["N"], c["C"]).to(t) if c["residual"] else None
        st["d_y"] = normal(c["N"], c["C"]).to(t)
        st["seed"] = (seed * 0x2545F4914F6CDD1D + 12345) & WORD
        st["offset"] = (seed * 7919) % (1 << 40)
    else:
        B, S = c["B"], c["S"]
        st["q"] = (1.5 * normal(B, c["Lq"], c["Hq"], c["D"])).to(t)
        st["kp"] = normal(c["P"], c["Hkv"], c["D"]).to(t)
        st["vp"] = normal(c["P"], c["Hkv"], c["D"]).to(t)
        st["ks"] = st["vs"] = st["n"] = None
        if S:
            st["ks"] = normal(B, S, c["Hkv"], c["D"]).to(t)
            st["vs"] = normal(B, S, c["Hkv"], c["D"]).to(t)
            st["n"] = torch.randint(0, S + 1, (B,), device=dev, generator=g, dtype=torch.int32)
            st["n"][-1] = S
            if B > 1:
                st["n"][0] = 0                             # a row without a suffix
    return st


# ------------------------------------------------------------------------------------------------------------ plain forms
def _doubling(a, b):
    """Inclusive scan of the maps h -> a h + b along dim 1.  Doubling, not cumulative products: those underflow within a
    few hundred steps, so that a quotient of two of them says nothing; the loop is over the logarithm of the length."""
    d = 1
    while d < a.shape[1]:
        b = torch.cat([b[:, :d], b[:, d:] + a[:, d:] * b[:, :-d]], 1)
        a = torch.cat([a[:, :d], a[:, d:] * a[:, :-d]], 1)
        d *= 2
    return a, b


def _gates(z, v, begin):
    z, v = z.float(), v.float()
    a, u = 1.0 / (1.0 + torch.exp(-z)), 1.0 / (1.0 + torch.exp(z))
    if begin is None:
        return a, u, v, None
    live = (torch.arange(z.shape[1], device=z.device)[None, :] >= begin[:, None].long())[..., None]
    zero = torch.zeros((), device=z.device)
    return torch.where(live, a, zero + 1.0), torch.where(live, u, zero), torch.where(live, v, zero), live


def _plain_scan(st):
    C, p = st["C"], st["period"]
    z, v = st["proj"][..., :C], st["proj"][..., C:]
    a, u, v, live = _gates(z, v, st["begin"])
    start = st["start"] if st["start"] is not None else torch.zeros(a.shape[0], C, device=a.device)
    A, h = _doubling(a, u * v)
    h = h + A * start[:, None]
    y, h_last = h[:, p - 1::p].to(z.dtype), h[:, -1].clone()
    if not st["train"]:
        return {"y": y, "h_last": h_last}
    d = torch.zeros_like(h)
    d[:, p - 1::p] = st["d_y"].float()
    d[:, -1] += st["d_h_last"]
    after = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)        # a of the step behind
    _, G = _doubling(after.flip(1), d.flip(1))
    G = G.flip(1)
    before = torch.cat([start[:, None], h[:, :-1]], 1)
    d_v, d_z = u * G, G * (before - v) * a * u
    if live is not None:
        zero = torch.zeros((), device=z.device)
        d_v, d_z = torch.where(live, d_v, zero), torch.where(live, d_z, zero)
    return {"y": y, "h_last": h_last, "d_z": d_z.to(z.dtype), "d_v": d_v.to(z.dtype), "d_h0": a[:, 0] * G[:, 0]}


def _plain_step(st):
    z, v, h = st["z"].float(), st["v"].float(), st["store"][st["user"].long()]
    a, u = 1.0 / (1.0 + torch.exp(-z)), 1.0 / (1.0 + torch.exp(z))
    return (a * h + u * v).to(st["z"].dtype)


def _signed(x):
    """A 64-bit word as torch's int64 holds it."""
    x &= WORD
    return x - (1 << 64) if x >> 63 else x


def _right(x, n):
    return (x >> n) & ((1 << (64 - n)) - 1)


def _mix(x):
    x = (x ^ _right(x, 30)) * _signed(MIX1)
    x = (x ^ _right(x, 27)) * _signed(MIX2)
    return x ^ _right(x, 31)


def _mix_word(x):
    x = ((x ^ (x >> 30)) * MIX1) & WORD
    x = ((x ^ (x >> 27)) * MIX2) & WORD
    return x ^ (x >> 31)


def _kept(n, keep, seed, offset, dev):
    """Element i is kept where 16-bit field i % 4 of word i // 4 is below keep * 65536; word k is the splitmix64 output of
    counter offset + k under the mixed seed."""
    i = torch.arange((n + 3) // 4, device=dev)
    word = _mix((i + (_signed(offset) + 1)) * _signed(GOLDEN) + _signed(_mix_word(seed)))
    field = torch.stack([_right(word, 16 * j) & 0xFFFF if j else word & 0xFFFF for j in range(4)], 1).reshape(-1)[:n]
    return field < _threshold(keep)


def _threshold(keep):
    return min(65536, max(1, int(math.floor(keep * 65536 + 0.5))))


def _plain_dropout(st):
    x, d = st["x"], st["d_y"]
    kept = _kept(x.numel(), st["keep"], st["seed"], st["offset"], x.device).reshape(x.shape)
    scale = 65536.0 / _threshold(st["keep"])
    zero = torch.zeros((), device=x.device)
    y = torch.where(kept, x.float() * scale, zero)
    if st["res"] is not None:
        y = y + st["res"].float()
    return {"y": y.to(x.dtype), "d_x": torch.where(kept, d.float() * scale, zero).to(x.dtype)}


def _plain_attn(st):
    q, B, Lq, Hq, Hkv, D, S = st["q"], st["B"], st["Lq"], st["Hq"], st["Hkv"], st["D"], st["S"]
    G = Hq // Hkv
    qh = q.float().reshape(B, Lq, Hkv, G, D) * (1.0 / math.sqrt(D))
    rows = qh.permute(2, 0, 1, 3, 4).reshape(Hkv, B * Lq * G, D)
    sp = torch.bmm(rows, st["kp"].float().permute(1, 2, 0).contiguous())                       # [Hkv, rows, P]
    m = sp.amax(-1)
    if S:
        of_row = qh.permute(0, 2, 1, 3, 4).reshape(B * Hkv, Lq * G, D)
        ss = torch.bmm(of_row, st["ks"].float().permute(0, 2, 3, 1).reshape(B * Hkv, D, S).contiguous()).reshape(B, Hkv, Lq, G, S)
        # query token i of a row's last Lq tokens sees the suffix up to its own position
        sees = st["n"].long()[:, None] - Lq + 1 + torch.arange(Lq, device=q.device)[None, :]
        seen = torch.arange(S, device=q.device)[None, None, :] < sees[..., None]
        ss = torch.where(seen[:, None, :, None, :], ss, torch.full((), -math.inf, device=q.device))
        ms = ss.amax(-1).permute(1, 0, 2, 3).reshape(Hkv, B * Lq * G)
        m = torch.maximum(m, ms)
    sp = torch.exp(sp - m[..., None])
    total = sp.sum(-1)
    out = torch.bmm(sp, st["vp"].float().permute(1, 0, 2).contiguous())
    if S:
        ps = torch.exp(ss - m.reshape(Hkv, B, Lq, G).permute(1, 0, 2, 3)[..., None])
        total = total + ps.sum(-1).permute(1, 0, 2, 3).reshape(Hkv, -1)
        vs = st["vs"].float().permute(0, 2, 1, 3).reshape(B * Hkv, S, D).contiguous()
        out = out + torch.bmm(ps.reshape(B * Hkv, Lq * G, S), vs).reshape(B, Hkv, Lq * G, D).permute(1, 0, 2, 3).reshape(Hkv, -1, D)
    out = (out / total[..., None]).reshape(Hkv, B, Lq, G, D).permute(1, 2, 0, 3, 4).reshape(B, Lq, Hq, D).to(q.dtype)
    if not st["lse"]:
        return out
    return {"out": out, "lse": (m + torch.log(total)).reshape(Hkv, B, Lq, G).permute(1, 2, 0, 3).reshape(B, Lq, Hq)}


# ---------------------------------------------------------------------------------------------------------------- one pass
def run(st):
    if not own:
        return {"scan": _plain_scan, "step": _plain_step, "dropout": _plain_dropout, "attn": _plain_attn}[st["op"]](st)
    from hpmn_amd import ops
    if st["op"] == "scan":
        z, v = st["proj"][..., :st["C"]], st["proj"][..., st["C"]:]
        y, h_last, saved = ops.gated_scan_fwd(z, v, h0=st["start"], begin=st["begin"], period=st["period"], train=st["train"])
        if not st["train"]:
            return {"y": y, "h_last": h_last}
        d_z, d_v, d_h0 = ops.gated_scan_bwd(z, v, saved, st["d_y"], d_h_last=st["d_h_last"], begin=st["begin"], period=st["period"])
        return {"y": y, "h_last": h_last, "d_z": d_z, "d_v": d_v, "d_h0": d_h0}
    if st["op"] == "step":
        return ops.gated_scan_step(st["z"], st["v"], st["store"], user=st["user"], commit=False)
    if st["op"] == "dropout":
        y = ops.dropout_fwd(st["x"], st["keep"], st["seed"], offset=st["offset"], residual=st["res"])
        return {"y": y, "d_x": ops.dropout_bwd(st["d_y"], st["keep"], st["seed"], offset=st["offset"])}
    got = ops.shared_prefix_attention(st["q"], st["kp"], st["vp"], st["ks"], st["vs"], suffix_len=st["n"], want_lse=st["lse"])
    return {"out": got[0], "lse": got[1]} if st["lse"] else got


# --------------------------------------------------------------------------------------------------------------- in 64 bits
def exact(c, seed):
    st = prepare(c, seed)
    f = torch.float64
    if c["op"] == "scan":
        B, T, C, p = c["B"], c["T"], c["C"], c["period"]
        z, v = st["proj"][..., :C], st["proj"][..., C:]
        begin = st["begin"].long() if c["pad"] else torch.zeros(B, device=z.device, dtype=torch.long)
        h = st["start"].to(f) if c["h0"] else torch.zeros(B, C, device=z.device, dtype=f)
        first, ys, states = h, [], []
        for t in range(T):                                 # the recurrence as it is written
            a = torch.sigmoid(z[:, t].to(f))
            new = a * h + torch.sigmoid(-z[:, t].to(f)) * v[:, t].to(f)
            h = torch.where((begin <= t)[:, None], new, h) if c["pad"] else new
            if c["train"]:
                states.append(h)
            if (t + 1) % p == 0:
                ys.append(h)
        got = {"y": torch.stack(ys, 1), "h_last": h}
        if not c["train"]:
            return got
        d_z, d_v = torch.empty(B, T, C, device=z.device, dtype=f), torch.empty(B, T, C, device=z.device, dtype=f)
        d = st["d_h_last"].to(f)
        for t in range(T - 1, -1, -1):
            if (t + 1) % p == 0:
                d = d + st["d_y"][:, t // p].to(f)
            a, u = torch.sigmoid(z[:, t].to(f)), torch.sigmoid(-z[:, t].to(f))
            there = (begin <= t)[:, None]
            d_v[:, t] = torch.where(there, u * d, 0.0)
            d_z[:, t] = torch.where(there, a * u * (states[t - 1] if t else first).sub(v[:, t].to(f)) * d, 0.0)
            d = torch.where(there, a * d, d)
        return {**got, "d_z": d_z, "d_v": d_v, "d_h0": d}
    if c["op"] == "step":
        z = st["z"].to(f)
        return torch.sigmoid(z) * st["store"][st["user"].long()].to(f) + torch.sigmoid(-z) * st["v"].to(f)
    if c["op"] == "dropout":
        n = c["N"] * c["C"]
        # the same words from numpy's unsigned 64-bit arithmetic
        import numpy as np
        with np.errstate(over="ignore"):
            k = np.arange((n + 3) // 4, dtype=np.uint64) + np.uint64(st["offset"] + 1)
            w = k * np.uint64(GOLDEN) + np.uint64(_mix_word(st["seed"]))
            w = (w ^ (w >> np.uint64(30))) * np.uint64(MIX1)
            w = (w ^ (w >> np.uint64(27))) * np.uint64(MIX2)
            w ^= w >> np.uint64(31)
        keep = w.astype("<u8").view("<u2")[:n] < _threshold(c["keep"]) if c["keep"] < 1 else np.ones(n, bool)
        m = torch.from_numpy(keep).to(st["x"].device).reshape(c["N"], c["C"]).to(f) * (65536.0 / _threshold(c["keep"]))
        y = st["x"].to(f) * m
        return {"y": y + st["res"].to(f) if c["residual"] else y, "d_x": st["d_y"].to(f) * m}
    B, Lq, Hq, Hkv, D = c["B"], c["Lq"], c["Hq"], c["Hkv"], c["D"]
    out = torch.empty(B, Lq, Hq, D, device=st["q"].device, dtype=f)
    lse = torch.empty(B, Lq, Hq, device=st["q"].device, dtype=f)
    for h in range(Hq):
        k = h // (Hq // Hkv)
        q = st["q"][:, :, h].to(f) / math.sqrt(D)                                              # [B, Lq, D]
        s = q.reshape(-1, D) @ st["kp"][:, k].to(f).t().contiguous()
        l, o = torch.logsumexp(s, -1), torch.softmax(s, -1) @ st["vp"][:, k].to(f)
        l, o = l.reshape(B, Lq), o.reshape(B, Lq, D)
        if c["S"]:
            s = torch.bmm(q, st["ks"][:, :, k].to(f).transpose(1, 2).contiguous())             # [B, Lq, S]
            ends = st["n"].long()[:, None] - Lq + torch.arange(Lq, device=q.device)[None]
            s = s.masked_fill(torch.arange(c["S"], device=q.device)[None, None] > ends[..., None], -math.inf)
            both = torch.logaddexp(l, torch.logsumexp(s, -1))
            o = o * torch.exp(l - both)[..., None] + torch.bmm(torch.exp(s - both[..., None]), st["vs"][:, :, k].to(f).contiguous())
            l = both
        out[:, :, h], lse[:, :, h] = o, l
    return {"out": out, "lse": lse} if c["lse"] else out
