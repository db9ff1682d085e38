"""The operators of a token model's training step that are measured one by one, and how a program calls them.

A case's "op" names the operator:

    embed    embedding lookup with a scale (and positions), and the table's gradient from sorted tokens
    dropout  dropout (added to a residual) whose mask comes from a counter and is never stored, and its backward pass
    qknorm   RMS norm of every query and key head with the position rotation, and its backward pass
    gated    act(x Wg) * (x Wu) of a gated feed-forward layer, and its backward pass

"train" says whether the backward pass runs too.  All tensors are float32, as everywhere in this framework, and the
products run in its default precision.
"""
from __future__ import annotations

import math
import threading

import numpy as np
import torch

own = False

EPS = 1e-6
BASE = 10000.0


def listed():
    return [
        # The language-model configuration: 32 sequences of 128 tokens, vocabulary 1000, positions added.
        {"name": "embed_lm", "op": "embed", "tokens": 4096, "seq": 128, "dim": 256, "vocab": 1000, "skew": 0.0, "train": True},
        # A subword vocabulary: most rows get no token of the batch, a few get very many.
        {"name": "embed_subwords", "op": "embed", "tokens": 16384, "seq": 0, "dim": 1024, "vocab": 50000, "skew": 1.0, "train": True},
        # The lookup of a handful of tokens that are being generated, rows of an odd width.
        {"name": "embed_step", "op": "embed", "tokens": 9, "seq": 0, "dim": 999, "vocab": 32000, "skew": 0.0, "train": False},
        # The language-model configuration's activations behind a block: residual + dropout(x).
        {"name": "dropout_lm", "op": "dropout", "count": 32 * 128 * 256, "residual": True, "p": 0.1, "train": True},
        # The wide layer at its global batch of 16384, dropped on the way to the next one.
        {"name": "dropout_wide", "op": "dropout", "count": 16384 * 4096, "residual": False, "p": 0.5, "train": True},
        # The language-model configuration's heads: 8 of 32 features, one position per place in the sequence.
        {"name": "qknorm_lm", "op": "qknorm", "tokens": 4096, "seq": 128, "heads_q": 8, "heads_k": 8, "d_head": 32, "rot": 32,
         "interleaved": False, "far": 0, "train": True},
        # Long sequences, grouped heads in a packed projection.
        {"name": "qknorm_long", "op": "qknorm", "tokens": 16384, "seq": 8192, "heads_q": 32, "heads_k": 8, "d_head": 128, "rot": 128,
         "interleaved": False, "far": 0, "train": True},
        # Fifteen sequences that grow by a token each, far into their contexts; half of the features rotate.
        {"name": "qknorm_step", "op": "qknorm", "tokens": 15, "seq": 0, "heads_q": 16, "heads_k": 4, "d_head": 64, "rot": 32,
         "interleaved": True, "far": 100000, "train": False},
        # The language-model configuration's feed-forward, gated.
        {"name": "gated_lm", "op": "gated", "m": 4096, "k": 256, "n": 1024, "act": "gelu", "train": True},
        # A wide layer whose inner width is no power of two.
        {"name": "gated_wide", "op": "gated", "m": 8192, "k": 2048, "n": 5504, "act": "silu", "train": True},
        # An odd number of rows and odd widths, as a padded batch gives them.
        {"name": "gated_ragged", "op": "gated", "m": 1001, "k": 500, "n": 1333, "act": "silu", "train": True},
        # Three tokens that are being generated: the weights are read once.
        {"name": "gated_step", "op": "gated", "m": 3, "k": 1024, "n": 2752, "act": "silu", "train": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embed", "dropout", "qknorm", "gated"])
    if op == "embed":
        dim, vocab = rng.choice([64, 200, 256, 512, 777, 1000, 1024]), _log_int(rng, 100, 50000)
        train = rng.random() < 0.8
        tokens = _log_int(rng, 256, 16384) if train else _log_int(rng, 1, 16384)
        return {"op": "embed", "tokens": tokens, "seq": rng.choice([0, 128]), "dim": dim, "vocab": vocab, "skew": rng.choice([0.0, 0.8, 1.0]), "train": train}
    if op == "dropout":
        return {"op": "dropout", "count": _log_int(rng, 1000, 16384 * 4096), "residual": rng.random() < 0.5, "p": rng.choice([0.05, 0.1, 0.3, 0.5]),
                "train": rng.random() < 0.8}
    if op == "qknorm":
        d_head = rng.choice([32, 64, 80, 96, 128, 128, 256])
        heads_k = rng.choice([1, 2, 4, 8])
        heads_q = heads_k * rng.choice([1, 2, 4])
        train = rng.random() < 0.7
        most = 16384 * 40 * 128 // ((heads_q + heads_k) * d_head)
        tokens = min(most, _log_int(rng, 64, 16384) if train else _log_int(rng, 1, 4096))
        return {"op": "qknorm", "tokens": tokens, "seq": rng.choice([0, 128, 2048]), "heads_q": heads_q, "heads_k": heads_k, "d_head": d_head,
                "rot": rng.choice([d_head, d_head, d_head // 2]), "interleaved": rng.random() < 0.3, "far": rng.choice([0, 5000, 100000]), "train": train}
    train = rng.random() < 0.7
    k, n = _log_int(rng, 64, 2048), _log_int(rng, 128, 5504)
    m = _log_int(rng, 100, 8192) if train else _log_int(rng, 1, 512)
    if rng.random() < 0.6:
        k, n = max(64, k // 64 * 64), max(128, n // 64 * 64)
    return {"op": "gated", "m": m, "k": k, "n": n, "act": rng.choice(["silu", "gelu"]), "train": train}


def work(case):
    if case["op"] == "embed":
        t, d, v = case["tokens"], case["dim"], case["vocab"]
        b = 4.0 * (min(t, v) * d + t + t * d + min(t, case["seq"]) * d)
        f = t * d * (2.0 if case["seq"] else 1.0)
        if case["train"]:
            b += 4.0 * (t * d + v * d)
            f += t * d
        return {"bytes": b, "flops": f}
    if case["op"] == "dropout":
        n = case["count"]
        return {"bytes": 4.0 * n * (2 + case["residual"] + (2 if case["train"] else 0)), "flops": n * (2.0 if case["train"] else 1.0)}
    if case["op"] == "qknorm":
        n = case["tokens"] * (case["heads_q"] + case["heads_k"]) * case["d_head"]
        return {"bytes": 4.0 * n * (4 if case["train"] else 2), "flops": n * (20.0 if case["train"] else 6.0)}
    m, k, n = case["m"], case["k"], case["n"]
    b = 4.0 * (m * k + 2 * k * n + m * n)
    f = 4.0 * m * k * n
    if case["train"]:
        b += 4.0 * (m * n + m * k + 2 * k * n)
        f += 8.0 * m * k * n
    return {"bytes": b, "flops": f}


# ------------------------------------------------------------------------------------------------ inputs

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def randn(*shape, std=1.0):
        return torch.randn(*shape, device="cuda", generator=gen) * std

    s = {"case": case}
    if case["op"] == "embed":
        t, d, v = case["tokens"], case["dim"], case["vocab"]
        s["weight"] = randn(v, d, std=0.5)
        u = torch.rand(t, device="cuda", generator=gen, dtype=torch.float64)
        if case["skew"]:   # how often words occur: the rank's power, ranks spread over the table
            p = torch.arange(1, v + 1, device="cuda", dtype=torch.float64).pow(-case["skew"]).cumsum(0)
            rank = torch.searchsorted(p, u * p[-1]).clamp(max=v - 1)
            s["ids"] = torch.randperm(v, device="cuda", generator=gen)[rank].to(torch.int32)
        else:
            s["ids"] = (u * v).long().clamp(max=v - 1).to(torch.int32)
        s["pos"] = randn(case["seq"], d) if case["seq"] else None
        s["scale"] = math.sqrt(d)
        s["g"] = randn(t, d, std=1e-2) if case["train"] else None
    elif case["op"] == "dropout":
        n = case["count"]
        s["x"] = randn(n)
        s["residual"] = randn(n) if case["residual"] else None
        s["g"] = randn(n, std=1e-2) if case["train"] else None
        s["key"], s["first"] = 0x9E3779B97F4A7C15 ^ int(seed), 1000 * int(seed) + (1 << 33)
    elif case["op"] == "qknorm":
        t, hq, hk, d, rot = case["tokens"], case["heads_q"], case["heads_k"], case["d_head"], case["rot"]
        s["packed"] = randn(t, (hq + 2 * hk) * d, std=1.5)          # [queries | keys | values] of a projection
        s["gamma_q"], s["gamma_k"] = 1.0 + randn(d, std=0.2), 1.0 + randn(d, std=0.2)
        length = max(case["far"] + t + 1, case["seq"], t)
        s["table"] = _rotations(torch.arange(length, device="cuda"), rot).to(torch.float32).contiguous()   # [length, rot / 2, (cos, sin)]
        if case["seq"] and not case["far"]:
            s["positions"], s["seq"] = None, case["seq"]
        else:
            at = torch.randint(0, length, (t,), device="cuda", generator=gen) if case["far"] else torch.arange(t, device="cuda")
            s["positions"], s["seq"] = at.to(torch.int32), t
        s["gq"], s["gk"] = (randn(t, hq * d, std=1e-2), randn(t, hk * d, std=1e-2)) if case["train"] else (None, None)
    else:
        m, k, n = case["m"], case["k"], case["n"]
        s["x"] = randn(m, k)
        s["wg"], s["wu"] = randn(k, n, std=1.0 / math.sqrt(k)), randn(k, n, std=1.0 / math.sqrt(k))
        s["dh"] = randn(m, n, std=1e-2) if case["train"] else None
    return s


def _rotations(positions, rot):
    """cos and sin of position * base^(-2i / rot), the angle in 64 bits."""
    freq = BASE ** (-torch.arange(0, rot, 2, device=positions.device, dtype=torch.float64) / rot)
    angle = positions.to(torch.float64)[:, None] * freq
    return torch.stack([angle.cos(), angle.sin()], dim=-1)


# ------------------------------------------------------------------------------------------------ plain forms

def run(state):
    op = state["case"]["op"]
    if own:
        return {"embed": _own_embed, "dropout": _own_dropout, "qknorm": _own_qknorm, "gated": _own_gated}[op](state)
    return {"embed": _embed, "dropout": _dropout, "qknorm": _qknorm, "gated": _gated}[op](state)


def _embed(s):
    ids, w = s["ids"].long(), s["weight"]
    y = w[ids] * s["scale"]
    if s["pos"] is not None:
        y = y + s["pos"][torch.arange(ids.numel(), device=ids.device) % s["pos"].shape[0]]
    if s["g"] is None:
        return {"y": y}
    # (a frequent token's row is a long sum)
    dw = torch.zeros(w.shape, device=w.device, dtype=torch.float64).index_add_(0, ids, s["g"].double() * s["scale"])
    return {"y": y, "dw": dw.float()}


def _philox_words(key, first, count):
    """`count` words of Philox-4x32-10 blocks first, first + 1, ... under a 64-bit key; 64-bit integers wrap as the products need."""
    at = torch.arange((count + 3) // 4, device="cuda", dtype=torch.int64) + first
    low = 0xFFFFFFFF
    c0, c1 = at & low, (at >> 32) & low
    c2, c3 = torch.zeros_like(c0), torch.zeros_like(c0)
    k0, k1 = key & low, (key >> 32) & low
    for _ in range(10):   # the generator's ten rounds
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((p1 >> 32) & low) ^ c1 ^ k0, p1 & low, ((p0 >> 32) & low) ^ c3 ^ k1, p0 & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack([c0, c1, c2, c3], dim=1).reshape(-1)[:count]


def _dropout(s):
    case = s["case"]
    p = torch.tensor(case["p"], device="cuda", dtype=torch.float32)
    u = (_philox_words(s["key"], s["first"], case["count"]) >> 8).float() * 2.0 ** -24
    mask = torch.where(u < p, torch.zeros_like(u), 1.0 / (1.0 - p))
    y = s["x"] * mask
    if s["residual"] is not None:
        y = y + s["residual"]
    return {"y": y} if s["g"] is None else {"y": y, "dx": s["g"] * mask}


def _heads(packed, first, heads, d):
    return packed[:, first * d:(first + heads) * d].reshape(packed.shape[0], heads, d)


def _halves(x, rot, interleaved):
    """The two members of each rotated pair."""
    return (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])


def _joined(a, b, x, rot, interleaved):
    r = torch.stack([a, b], dim=-1).flatten(-2) if interleaved else torch.cat([a, b], dim=-1)
    return torch.cat([r, x[..., rot:]], dim=-1)


def _positions(s):
    t = s["case"]["tokens"]
    return s["positions"].long() if s["positions"] is not None else torch.arange(t, device="cuda") % s["seq"]


def _qknorm(s):
    case = s["case"]
    t, hq, hk, d, rot, inter = (case[k] for k in ("tokens", "heads_q", "heads_k", "d_head", "rot", "interleaved"))
    cs = s["table"][_positions(s)][:, None]
    c, sn = cs[..., 0], cs[..., 1]

    def one(x, gamma, g):
        rstd = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        xhat = x * rstd
        z = xhat * gamma
        a, b = _halves(z, rot, inter)
        y = _joined(a * c - b * sn, a * sn + b * c, z, rot, inter)
        if g is None:
            return y.reshape(t, -1), None, None
        g = g.reshape(x.shape)
        a, b = _halves(g, rot, inter)
        dz = _joined(a * c + b * sn, b * c - a * sn, g, rot, inter)
        dxhat = dz * gamma
        dx = rstd * (dxhat - xhat * (dxhat * xhat).mean(-1, keepdim=True))
        return y.reshape(t, -1), dx.reshape(t, -1), (dz * xhat).sum((0, 1))

    yq, dq, dgq = one(_heads(s["packed"], 0, hq, d), s["gamma_q"], s["gq"])
    yk, dk, dgk = one(_heads(s["packed"], hq, hk, d), s["gamma_k"], s["gk"])
    if s["gq"] is None:
        return {"q": yq, "k": yk}
    return {"q": yq, "k": yk, "dq": dq, "dk": dk, "dgamma_q": dgq, "dgamma_k": dgk}


def _gated(s):
    act, x, wg, wu, dh = s["case"]["act"], s["x"], s["wg"], s["wu"], s["dh"]
    a, u = x @ wg, x @ wu
    if act == "silu":
        e = 1.0 / (1.0 + (-a).exp())
        f, df = a * e, e * (1.0 + a * (1.0 - e))
    else:   # GELU's tanh form
        th = torch.tanh(0.7978845608 * (a + 0.044715 * a * a * a))
        f = 0.5 * a * (1.0 + th)
        df = 0.5 * (1.0 + th) + 0.5 * a * (1.0 - th * th) * 0.7978845608 * (1.0 + 3.0 * 0.044715 * a * a)
    h = f * u
    if dh is None:
        return {"h": h}
    da, du = dh * u * df, dh * f
    return {"h": h, "dx": da @ wg.T + du @ wu.T, "dwg": x.T @ da, "dwu": x.T @ du}


# ------------------------------------------------------------------------------------------------ the framework's calls

_here = threading.local()   # (which stream is the current one goes by the thread, too)


def _framework():
    """The library and a context on the program's own stream, made once; the stream waits for the inputs made before."""
    if not hasattr(_here, "handle"):
        from neuralrs_b200 import _lib, cuda
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        torch.cuda.set_stream(stream)
        ctx = cuda.Context(torch.cuda.current_device())
        ctx.set_stream(stream.cuda_stream)
        _here.handle = [_lib.lib(), ctx, stream, _lib.check, {"gelu": _lib.ACT_GELU, "silu": _lib.ACT_SILU}]
    return _here.handle


def _p(t, at=0):
    return None if t is None else t.data_ptr() + 4 * at


def _own_embed(s):
    lib, ctx, _, check, _ = _framework()
    w, ids, pos, g = s["weight"], s["ids"], s["pos"], s["g"]
    t, (v, d) = ids.numel(), w.shape
    y = torch.empty(t, d, device="cuda")
    check(ctx.h, lib.nrs_embedding_scaled_fwd(ctx.h, _p(w), _p(ids), _p(pos), _p(y), t, pos.shape[0] if pos is not None else 1, d, v, s["scale"]))
    if g is None:
        return {"y": y}
    dw = torch.empty(v, d, device="cuda")
    nbytes = lib.nrs_embedding_sorted_workspace(t, d, v)
    ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    check(ctx.h, lib.nrs_embedding_sorted_bwd(ctx.h, _p(g), _p(ids), _p(dw), t, d, v, s["scale"], 0, _p(ws), nbytes))
    return {"y": y, "dw": dw}


def _own_dropout(s):
    lib, ctx, _, check, _ = _framework()
    x, n, p = s["x"], s["case"]["count"], s["case"]["p"]
    y = torch.empty_like(x)
    check(ctx.h, lib.nrs_dropout_fwd(ctx.h, _p(x), _p(s["residual"]), _p(y), n, 1, p, s["key"], s["first"]))
    if s["g"] is None:
        return {"y": y}
    dx = torch.empty_like(x)
    check(ctx.h, lib.nrs_dropout_bwd(ctx.h, _p(s["g"]), _p(dx), n, 1, p, s["key"], s["first"], 0))
    return {"y": y, "dx": dx}


def _own_qknorm(s):
    lib, ctx, _, check, _ = _framework()
    case, x, table, at = s["case"], s["packed"], s["table"], s["positions"]
    t, hq, hk, d, rot = (case[k] for k in ("tokens", "heads_q", "heads_k", "d_head", "rot"))
    ld, shape = x.shape[1], (t, s["seq"], hq, hk, d, rot, table.shape[0], int(case["interleaved"]), EPS)
    q, k = torch.empty(t, hq * d, device="cuda"), torch.empty(t, hk * d, device="cuda")
    check(ctx.h, lib.nrs_qk_norm_rotary_fwd(ctx.h, _p(x), ld, _p(x, hq * d), ld, _p(s["gamma_q"]), _p(s["gamma_k"]), _p(table), _p(at),
                                            _p(q), hq * d, _p(k), hk * d, *shape))
    if s["gq"] is None:
        return {"q": q, "k": k}
    dq, dk = torch.empty_like(q), torch.empty_like(k)
    dgq, dgk = torch.empty(d, device="cuda"), torch.empty(d, device="cuda")
    nbytes = lib.nrs_qk_norm_rotary_workspace(t, hq, hk, d)
    ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    check(ctx.h, lib.nrs_qk_norm_rotary_bwd(ctx.h, _p(s["gq"]), hq * d, _p(s["gk"]), hk * d, _p(x), ld, _p(x, hq * d), ld, _p(s["gamma_q"]),
                                            _p(s["gamma_k"]), _p(table), _p(at), _p(dq), hq * d, _p(dk), hk * d, _p(dgq), _p(dgk), *shape,
                                            0, 0, _p(ws), nbytes))
    return {"q": q, "k": k, "dq": dq, "dk": dk, "dgamma_q": dgq, "dgamma_k": dgk}


def _own_gated(s):
    lib, ctx, _, check, acts = _framework()
    x, wg, wu, dh = s["x"], s["wg"], s["wu"], s["dh"]
    (m, k), n, act = x.shape, wg.shape[1], acts[s["case"]["act"]]
    h = torch.empty(m, n, device="cuda")
    if dh is None:
        check(ctx.h, lib.nrs_gated_linear_fwd(ctx.h, _p(x), _p(wg), _p(wu), _p(h), None, None, m, n, k, act))
        return {"h": h}
    a, u = torch.empty_like(h), torch.empty_like(h)
    check(ctx.h, lib.nrs_gated_linear_fwd(ctx.h, _p(x), _p(wg), _p(wu), _p(h), _p(a), _p(u), m, n, k, act))
    dx, dwg, dwu = torch.empty_like(x), torch.empty_like(wg), torch.empty_like(wu)
    check(ctx.h, lib.nrs_gated_linear_bwd(ctx.h, _p(x), _p(wg), _p(wu), _p(a), _p(u), _p(dh), _p(dx), _p(dwg), _p(dwu), m, n, k, act, 0, 0))
    return {"h": h, "dx": dx, "dwg": dwg, "dwu": dwu}


# ------------------------------------------------------------------------------------------------ from the definitions, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"embed": _exact_embed, "dropout": _exact_dropout, "qknorm": _exact_qknorm, "gated": _exact_gated}[case["op"]](s)


def _exact_embed(s):
    ids = s["ids"].long()
    y = s["weight"].double().index_select(0, ids) * s["scale"]
    if s["pos"] is not None:
        reps = -(-ids.numel() // s["pos"].shape[0])
        y = y + s["pos"].double().repeat(reps, 1)[:ids.numel()]
    if s["g"] is None:
        return {"y": y}
    # sums of runs of equal tokens, as differences of running sums over the tokens in order of their ids
    ordered, at = torch.sort(ids, stable=True)
    run = torch.cat([torch.zeros(1, s["g"].shape[1], device="cuda", dtype=torch.float64), s["g"].double()[at].cumsum(0)])
    edges = torch.searchsorted(ordered, torch.arange(s["weight"].shape[0] + 1, device="cuda"))
    return {"y": y, "dw": (run[edges[1:]] - run[edges[:-1]]) * s["scale"]}


def _exact_dropout(s):
    n, key, first = s["case"]["count"], s["key"], s["first"]
    keep = np.empty((n + 3) // 4 * 4, bool)
    p = float(np.float32(s["case"]["p"]))
    m0, m1, low, half = np.uint64(0xD2511F53), np.uint64(0xCD9E8D57), np.uint64(0xFFFFFFFF), np.uint64(32)
    for lo in range(0, keep.size // 4, 1 << 18):
        at = np.arange(lo, min(keep.size // 4, lo + (1 << 18)), dtype=np.uint64) + np.uint64(first)
        x = [at & low, at >> half, np.zeros_like(at), np.zeros_like(at)]
        k = [key & 0xFFFFFFFF, (key >> 32) & 0xFFFFFFFF]
        for _ in range(10):
            a, b = m0 * x[0], m1 * x[2]
            x = [(b >> half) ^ x[1] ^ np.uint64(k[0]), b & low, (a >> half) ^ x[3] ^ np.uint64(k[1]), a & low]
            k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
        keep[4 * lo:4 * (lo + at.size)] = (np.stack(x, axis=1).reshape(-1) >> np.uint64(8)).astype(np.float64) / 2.0 ** 24 >= p
    mask = torch.from_numpy(keep[:n]).cuda().double() / (1.0 - p)
    y = s["x"].double() * mask
    if s["residual"] is not None:
        y = y + s["residual"].double()
    return {"y": y} if s["g"] is None else {"y": y, "dx": s["g"].double() * mask}


def _exact_qknorm(s):
    case = s["case"]
    t, hq, hk, d, rot = (case[k] for k in ("tokens", "heads_q", "heads_k", "d_head", "rot"))
    at = s["positions"].double() if s["positions"] is not None else torch.remainder(torch.arange(t, device="cuda"), s["seq"]).double()
    angle = at[:, None, None] * torch.exp(-math.log(BASE) * 2.0 / rot * torch.arange(rot // 2, device="cuda", dtype=torch.float64))
    spin = torch.polar(torch.ones_like(angle), angle)
    out = {}
    for name, first, heads, gamma, g in (("q", 0, hq, s["gamma_q"], s["gq"]), ("k", hq, hk, s["gamma_k"], s["gk"])):
        x = s["packed"][:, first * d:(first + heads) * d].double().reshape(t, heads, d).requires_grad_(g is not None)
        w = gamma.double().requires_grad_(g is not None)
        z = x / (x.square().sum(-1, keepdim=True) / d + EPS).sqrt() * w
        r = z[..., :rot]
        turned = torch.view_as_complex((r.unflatten(-1, (rot // 2, 2)) if case["interleaved"] else r.unflatten(-1, (2, rot // 2)).transpose(-1, -2)).contiguous()) * spin
        turned = torch.view_as_real(turned)
        turned = turned.flatten(-2) if case["interleaved"] else turned.transpose(-1, -2).flatten(-2)
        y = torch.cat([turned, z[..., rot:]], -1).reshape(t, heads * d)
        out[name] = y.detach()
        if g is not None:
            dx, dw = torch.autograd.grad(y, (x, w), g.double())
            out["d" + name], out["dgamma_" + name] = dx.reshape(t, heads * d), dw
    return out


def _exact_gated(s):
    train = s["dh"] is not None
    x, wg, wu = (s[k].double().requires_grad_(train) for k in ("x", "wg", "wu"))
    a = x @ wg
    if s["case"]["act"] == "silu":
        f = a * torch.sigmoid(a)
    else:   # x * (1 + tanh(v)) / 2 = x * sigmoid(2v)
        f = a * torch.sigmoid(2.0 * 0.7978845608 * (a + 0.044715 * a ** 3))
    h = f * (x @ wu)
    if not train:
        return {"h": h}
    dx, dwg, dwu = torch.autograd.grad(h, (x, wg, wu), s["dh"].double())
    return {"h": h.detach(), "dx": dx, "dwg": dwg, "dwu": dwu}
