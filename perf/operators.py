"""Attention and dropout as programs built on ugk use them, as cases to time and to check.

A case is a dict of plain values; its "kind" names what one pass is:

  attend    attention over whole prompts, causal, from rows that hold q, k and v side by side: out and lse
  decode    one query row (or a few) per sequence against a cache of keys and values of fixed capacity,
            filled to a length of its own: out and lse
  backward  the gradient of attend: dqkv, from the rows, the forward's out and lse, and dout
  dropout   dropout of a flat array (the embedding's) and its backward
  droplayer a block's residual add with dropout of the branch, and the LayerNorm behind it, then the
            backward of both

Sequences: B of T rows each ("lens" is "equal"), or packed one behind the other with lengths drawn from
"len_seed" ("ragged"). HS is the size of a head, NH and NKV the numbers of query and key/value heads.
Everything is fp32, as the framework's buffers are.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

P_DROP, SEED, STEP, SITE = 0.1, 0x5EED, 3, 2


def listed():
    return [
        # one block of the character-level model (4 x 64 tokens, 6 heads): a call of a few microseconds
        {"name": "attend_text8", "kind": "attend", "lens": "equal", "B": 4, "T": 64, "NH": 6, "NKV": 6, "HS": 64},
        # one block of GPT-2-124M at the step's batch
        {"name": "attend_gpt2", "kind": "attend", "lens": "equal", "B": 8, "T": 1024, "NH": 12, "NKV": 12, "HS": 64},
        # documents of different lengths packed into one batch, four query heads to a key/value head
        {"name": "attend_packed", "kind": "attend", "lens": "ragged", "B": 13, "rows": 8191, "len_seed": 5, "NH": 16,
         "NKV": 4, "HS": 128},
        # one long document
        {"name": "attend_long", "kind": "attend", "lens": "equal", "B": 1, "T": 16384, "NH": 12, "NKV": 12, "HS": 64},
        # the next token of 16 sequences of GPT-2-124M
        {"name": "decode_gpt2", "kind": "decode", "B": 16, "cap": 1024, "Q": 1, "len_seed": 3, "NH": 12, "NKV": 12,
         "HS": 64},
        # the next token of 24 long conversations, four query heads to a key/value head
        {"name": "decode_long", "kind": "decode", "B": 24, "cap": 16384, "Q": 1, "len_seed": 4, "NH": 32, "NKV": 8,
         "HS": 128},
        # the gradients of the first three
        {"name": "backward_text8", "kind": "backward", "lens": "equal", "B": 4, "T": 64, "NH": 6, "NKV": 6, "HS": 64},
        {"name": "backward_gpt2", "kind": "backward", "lens": "equal", "B": 8, "T": 1024, "NH": 12, "NKV": 12,
         "HS": 64},
        {"name": "backward_packed", "kind": "backward", "lens": "ragged", "B": 7, "rows": 4095, "len_seed": 6, "NH": 16,
         "NKV": 4, "HS": 64},
        # the character-level model's embedding: latency
        {"name": "dropout_text8", "kind": "dropout", "n": 4 * 64 * 384},
        # a block of GPT-2-124M at the step's batch
        {"name": "droplayer_gpt2", "kind": "droplayer", "B": 8, "T": 1024, "C": 768},
        # a wider one whose rows are no whole number of 16-byte groups, over sequences of odd length
        {"name": "droplayer_odd", "kind": "droplayer", "B": 3, "T": 1023, "C": 1602},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng, most):
    """(NH, NKV, HS): mostly heads of 64, now and then of 128, seldom of another size."""
    group = rng.choice((1, 1, 1, 2, 3, 4, 8))
    nkv = max(1, _log_int(rng, 1, most) // group)
    return nkv * group, nkv, rng.choice((64, 64, 64, 128, 128, 32, 80, 50))


def draw(rng):
    kind = rng.choice(("attend", "attend", "decode", "decode", "backward", "backward", "dropout", "droplayer"))
    if kind == "dropout":
        return {"kind": kind, "n": _log_int(rng, 1000, 30000000)}
    if kind == "droplayer":
        C = _log_int(rng, 64, 4096)
        C = max(8, C // 64 * 64 if rng.random() < 0.6 else C)
        rows = _log_int(rng, 64, min(16384, (1 << 23) // C))
        B = _log_int(rng, 1, max(1, min(16, rows // 32)))
        return {"kind": kind, "B": B, "T": max(1, min(1024, rows // B - rng.randrange(2))), "C": C}
    NH, NKV, HS = _heads(rng, 16)
    if kind == "decode":
        cap = _log_int(rng, 16, 16384)
        B = _log_int(rng, 1, max(1, min(64, (1 << 27) // (cap * NKV * HS))))
        return {"kind": kind, "B": B, "cap": cap, "Q": rng.choice((1, 1, 1, 2, 4)), "len_seed": rng.randrange(1000),
                "NH": NH, "NKV": NKV, "HS": HS}
    T = _log_int(rng, 16, 4096 if kind == "attend" else 2048)
    B = _log_int(rng, 1, max(1, min(32, (1 << 24) // (T * NH * HS))))
    T -= rng.randrange(2)
    if rng.random() < 0.5:
        return {"kind": kind, "lens": "equal", "B": B, "T": T, "NH": NH, "NKV": NKV, "HS": HS}
    return {"kind": kind, "lens": "ragged", "B": B, "rows": B * T, "len_seed": rng.randrange(1000), "NH": NH, "NKV": NKV,
            "HS": HS}


def _lengths(c):
    """The sequences' lengths (of the cache's filled part for decode)."""
    if c["kind"] == "decode":
        rng = random.Random(c["len_seed"])
        return [rng.randint(min(c["Q"], c["cap"]), c["cap"]) for _ in range(c["B"])]
    if c["lens"] == "equal":
        return [c["T"]] * c["B"]
    rng = random.Random(c["len_seed"])
    w = [math.exp(rng.uniform(0.0, 3.0)) for _ in range(c["B"])]
    lens = [max(1, int(c["rows"] * x / sum(w))) for x in w]
    lens[lens.index(max(lens))] += c["rows"] - sum(lens)
    return lens


# ---- inputs ---------------------------------------------------------------------

def _rand(g, *shape, scale=1.0, mean=0.0):
    t = torch.randn(*shape, generator=g, device="cuda")
    if scale != 1.0:
        t.mul_(scale)
    return t.add_(mean) if mean else t


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    c, kind = case, case["kind"]
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    if kind == "dropout":
        n = c["n"]
        return {"case": c, "seed": SEED + seed, "inp": _rand(g, n), "dout": _rand(g, n),
                "out": torch.empty(n, device="cuda"), "dinp": torch.empty(n, device="cuda")}
    if kind == "droplayer":
        rows, C = c["B"] * c["T"], c["C"]
        e = lambda *s: torch.empty(*s, device="cuda")  # noqa: E731
        # dres: the gradient of res that the block above left
        return {"case": c, "seed": SEED + seed, "x": _rand(g, rows, C), "y": _rand(g, rows, C),
                "weight": _rand(g, C, scale=0.1, mean=1.0), "bias": _rand(g, C, scale=0.1), "dout": _rand(g, rows, C),
                "dres": _rand(g, rows, C), "res": e(rows, C), "out": e(rows, C), "mean": e(rows), "rstd": e(rows),
                "dinp": e(rows, C), "dx": e(rows, C), "dy": e(rows, C), "dparam": e(2, C)}
    NH, NKV, HS, lens = c["NH"], c["NKV"], c["HS"], _lengths(c)
    s = {"case": c, "scale": 1.0 / math.sqrt(HS)}
    if kind == "decode":
        B, cap, Q = c["B"], c["cap"], c["Q"]
        rows = B * Q
        s["q"] = _rand(g, rows, NH * HS)
        s["k"], s["v"] = _rand(g, B * cap, NKV * HS), _rand(g, B * cap, NKV * HS)
        s["q_start"] = _ints([b * Q for b in range(B)])
        s["q_end"] = _ints([(b + 1) * Q for b in range(B)])
        s["k_start"] = _ints([b * cap for b in range(B)])
        s["k_end"] = _ints([b * cap + n for b, n in enumerate(lens)])
        s["max_q"], s["max_k"] = Q, cap
    else:
        rows = sum(lens)
        s["qkv"] = _rand(g, rows, (NH + 2 * NKV) * HS)
        start = [sum(lens[:b]) for b in range(len(lens) + 1)]
        s["cu"] = _ints(start)
        s["q_start"] = s["k_start"] = s["cu"][:-1]
        s["q_end"] = s["k_end"] = s["cu"][1:]
        s["max_q"] = s["max_k"] = max(lens)
    s["out"], s["lse"] = torch.empty(rows, NH * HS, device="cuda"), torch.empty(rows, NH, device="cuda")
    if kind == "backward":
        s["dout"] = _rand(g, rows, NH * HS)
        o, l = _attend(s, c)  # the forward's results, which a training step has at this point
        s["out"].copy_(o)
        s["lse"].copy_(l)
        s["dqkv"] = torch.empty_like(s["qkv"])
    return s


# ---- one pass -------------------------------------------------------------------

def run(s):
    return (_OWN if own else _PLAIN)[s["case"]["kind"]](s, s["case"])


def _ugk():
    path = os.path.join(os.getcwd(), "uncertain-gpt_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import ugk
    return ugk


def _shape(ugk, s, c):
    """The call's sequences, heads and row strides."""
    NH, NKV, HS = c["NH"], c["NKV"], c["HS"]
    equal = c.get("lens") == "equal"
    ld = {} if c["kind"] == "decode" else {"ldq": (NH + 2 * NKV) * HS, "ldk": (NH + 2 * NKV) * HS,
                                           "ldv": (NH + 2 * NKV) * HS}
    seqs = {} if equal else {k: s[k] for k in ("q_start", "q_end", "k_start", "k_end")}
    rows_q = s["out"].shape[0]
    rows_k = s["k"].shape[0] if c["kind"] == "decode" else rows_q
    return ugk.Attention(nseq=c["B"], NH=NH, NKV=NKV, HS=HS, rows_q=rows_q, rows_k=rows_k, max_q=s["max_q"],
                         max_k=s["max_k"], causal=True, scale=s["scale"], **ld, **seqs)


def _split(s, c, t):
    """q, k and v where they start in rows that hold them side by side."""
    if c["kind"] == "decode":
        return s["q"], s["k"], s["v"]
    flat, NH, NKV, HS = t.view(-1), c["NH"], c["NKV"], c["HS"]
    return flat, flat[NH * HS:], flat[(NH + NKV) * HS:]


def _own_attend(s, c):
    ugk = _ugk()
    q, k, v = _split(s, c, s.get("qkv"))
    ugk.attention_forward(s["out"], s["lse"], q, k, v, _shape(ugk, s, c))
    return {"out": s["out"], "lse": s["lse"]}


def _own_backward(s, c):
    ugk = _ugk()
    q, k, v = _split(s, c, s["qkv"])
    dq, dk, dv = _split(s, c, s["dqkv"])
    ugk.attention_backward_zeroed(dq, dk, dv, s["dout"], q, k, v, s["out"], s["lse"], _shape(ugk, s, c))
    return {"dqkv": s["dqkv"]}


def _own_dropout(s, c):
    ugk = _ugk()
    n = c["n"]
    ugk.dropout_forward(s["out"], s["inp"], n, P_DROP, s["seed"], STEP, SITE)
    s["dinp"].zero_()  # backward outputs accumulate
    ugk.dropout_backward(s["dinp"], s["dout"], n, P_DROP, s["seed"], STEP, SITE)
    return {"out": s["out"], "dinp": s["dinp"]}


def _own_droplayer(s, c):
    ugk = _ugk()
    B, T, C = c["B"], c["T"], c["C"]
    drop = (P_DROP, s["seed"], STEP, SITE)
    ugk.dropout_residual_layernorm_forward(s["res"], s["out"], s["mean"], s["rstd"], s["x"], s["y"], s["weight"], s["bias"],
                                           B, T, C, *drop)
    s["dinp"].copy_(s["dres"])  # backward outputs accumulate: onto the gradient from above, and onto zeros
    for k in ("dx", "dy", "dparam"):
        s[k].zero_()
    ugk.layernorm_dropout_residual_backward(s["dinp"], s["dparam"][0], s["dparam"][1], s["dx"], s["dy"], s["dout"], s["res"],
                                            s["weight"], s["mean"], s["rstd"], B, T, C, *drop)
    return {k: s[k] for k in ("res", "out", "mean", "rstd", "dinp", "dx", "dy", "dparam")}


_OWN = {"attend": _own_attend, "decode": _own_attend, "backward": _own_backward, "dropout": _own_dropout,
        "droplayer": _own_droplayer}


def _padded(s, c):
    """Row numbers of q and k, (B, longest), their truth values, and the allowed pairs, (B, longest q, longest k)."""
    i = torch.arange(s["max_q"], device="cuda")
    j = torch.arange(s["max_k"], device="cuda")
    qs, qe, ks, ke = (s[k].long()[:, None] for k in ("q_start", "q_end", "k_start", "k_end"))
    in_q, in_k = i < qe - qs, j < ke - ks
    at_q, at_k = torch.where(in_q, qs + i, 0), torch.where(in_k, ks + j, 0)
    shift = ((ke - ks) - (qe - qs))[:, :, None]
    return at_q, at_k, in_q, in_k[:, None, :] & in_q[:, :, None] & (j <= i[:, None] + shift)


def _three(s, c):
    """q, k and v as (rows, heads, HS)."""
    NH, NKV, HS = c["NH"], c["NKV"], c["HS"]
    if c["kind"] == "decode":
        return s["q"].view(-1, NH, HS), s["k"].view(-1, NKV, HS), s["v"].view(-1, NKV, HS)
    t = s["qkv"].view(-1, NH + 2 * NKV, HS)
    return t[:, :NH], t[:, NH:NH + NKV], t[:, NH + NKV:]


def _grouped(t, at, NKV):
    """(rows, NH, HS) as (B, NKV, NH/NKV, longest, HS)."""
    B, T = at.shape
    return t[at].view(B, T, NKV, -1, t.shape[2]).permute(0, 2, 3, 1, 4).contiguous()


def _attend(s, c):
    NH, NKV, HS = c["NH"], c["NKV"], c["HS"]
    q, k, v = _three(s, c)
    at_q, at_k, in_q, ok = _padded(s, c)
    Q, K, V = _grouped(q, at_q, NKV), _grouped(k, at_k, NKV), _grouped(v, at_k, NKV)
    S = torch.matmul(Q, K.transpose(3, 4)).mul_(s["scale"])
    S.masked_fill_(~ok[:, None, None], float("-inf"))
    m = S.amax(4, keepdim=True)
    m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    P = S.sub_(m).exp_()
    l = P.sum(4, keepdim=True)
    O = torch.matmul(P, V) / torch.where(l == 0, torch.ones_like(l), l)
    lse = (m + torch.log(l)).squeeze(4)
    rows = at_q[in_q]
    out, stat = torch.zeros_like(s["out"]), torch.zeros_like(s["lse"])
    out[rows] = O.permute(0, 3, 1, 2, 4).reshape(len(at_q), -1, NH * HS)[in_q]
    stat[rows] = lse.permute(0, 3, 1, 2).reshape(len(at_q), -1, NH)[in_q]
    return out, stat


def _plain_attend(s, c):
    out, lse = _attend(s, c)
    return {"out": out, "lse": lse}


def _plain_backward(s, c):
    NH, NKV, HS = c["NH"], c["NKV"], c["HS"]
    q, k, v = _three(s, c)
    at_q, at_k, in_q, ok = _padded(s, c)
    Q, K, V = _grouped(q, at_q, NKV), _grouped(k, at_k, NKV), _grouped(v, at_k, NKV)
    dO = _grouped(s["dout"].view(-1, NH, HS), at_q, NKV)
    O = _grouped(s["out"].view(-1, NH, HS), at_q, NKV)
    L = s["lse"][at_q].view(len(at_q), -1, NKV, NH // NKV).permute(0, 2, 3, 1)[..., None]
    P = torch.matmul(Q, K.transpose(3, 4)).mul_(s["scale"]).sub_(L).exp_().masked_fill_(~ok[:, None, None], 0.0)
    dV = torch.matmul(P.transpose(3, 4), dO).sum(2)
    dS = torch.matmul(dO, V.transpose(3, 4)).sub_((dO * O).sum(4, keepdim=True)).mul_(P).mul_(s["scale"])
    dQ = torch.matmul(dS, K)
    dK = torch.matmul(dS.transpose(3, 4), Q).sum(2)
    dqkv = torch.zeros_like(s["qkv"]).view(-1, NH + 2 * NKV, HS)
    rows, B = at_q[in_q], len(at_q)
    dqkv[rows, :NH] = dQ.permute(0, 3, 1, 2, 4).reshape(B, -1, NH, HS)[in_q]
    dqkv[rows, NH:NH + NKV] = dK.permute(0, 2, 1, 3)[in_q]
    dqkv[rows, NH + NKV:] = dV.permute(0, 2, 1, 3)[in_q]
    return {"dqkv": dqkv.view_as(s["qkv"])}


def _philox_keep(n, p, seed, step, site):
    """Which of n elements stay: word i % 4 of Philox4x32-10 at counter {i / 4, step, 1 + site} is at least p 2^32."""
    low = 0xFFFFFFFF
    i = torch.arange((n + 3) // 4, device="cuda", dtype=torch.int64)
    c0, c1, c2, c3 = i & low, i >> 32, torch.full_like(i, step & low), torch.full_like(i, 1 + site)
    k0, k1 = seed & low, seed >> 32 & low
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (b >> 32 & low) ^ c1 ^ k0, b & low, (a >> 32 & low) ^ c3 ^ k1, a & low
        k0, k1 = k0 + 0x9E3779B9 & low, k1 + 0xBB67AE85 & low
    return torch.stack((c0, c1, c2, c3), 1).view(-1)[:n] >= round(p32(p) * 2 ** 32)


def p32(p):
    """p as a 32-bit float holds it."""
    return float(np.float32(p))


def _drop(t, keep):
    return torch.where(keep, t * (1.0 / (1.0 - p32(P_DROP))), torch.zeros_like(t))


def _plain_dropout(s, c):
    keep = _philox_keep(c["n"], P_DROP, s["seed"], STEP, SITE)
    return {"out": _drop(s["inp"], keep), "dinp": _drop(s["dout"], keep)}


def _plain_droplayer(s, c):
    rows, C = s["x"].shape
    keep = _philox_keep(rows * C, P_DROP, s["seed"], STEP, SITE).view(rows, C)
    res = s["x"] + _drop(s["y"], keep)
    mean = res.mean(1, keepdim=True)
    rstd = 1.0 / ((res - mean).square().mean(1, keepdim=True) + 1e-5).sqrt()
    xhat = (res - mean) * rstd
    dn = s["dout"] * s["weight"]
    dinp = s["dres"] + rstd * (dn - dn.mean(1, keepdim=True) - xhat * (dn * xhat).mean(1, keepdim=True))
    return {"res": res, "out": xhat * s["weight"] + s["bias"], "mean": mean.view(-1), "rstd": rstd.view(-1), "dinp": dinp,
            "dx": dinp, "dy": _drop(dinp, keep), "dparam": torch.stack(((s["dout"] * xhat).sum(0), s["dout"].sum(0)))}


_PLAIN = {"attend": _plain_attend, "decode": _plain_attend, "backward": _plain_backward, "dropout": _plain_dropout,
          "droplayer": _plain_droplayer}


# ---- what a pass cannot do without -------------------------------------------------

def work(case):
    """Bytes with each input read once and each output written once, and the float operations."""
    c, kind = case, case["kind"]
    if kind == "dropout":  # inp, dout read; out, dinp written
        return {"bytes": 16 * c["n"], "flops": 4 * c["n"]}
    if kind == "droplayer":  # x, y, dout, dres read; res, out, dinp, dx, dy written; res read again by the backward
        N = c["B"] * c["T"] * c["C"]
        return {"bytes": 40 * N + 16 * c["B"] * c["T"] + 20 * c["C"], "flops": 30 * N}
    NH, NKV, HS, lens = c["NH"], c["NKV"], c["HS"], _lengths(c)
    if kind == "decode":
        Q = c["Q"]
        pairs = sum(Q * n - Q * (Q - 1) // 2 for n in lens)
        return {"bytes": 4 * (2 * c["B"] * Q * NH * HS + c["B"] * Q * NH + 2 * sum(lens) * NKV * HS),
                "flops": 4 * pairs * NH * HS}
    rows, pairs = sum(lens), sum(n * (n + 1) // 2 for n in lens)
    qkv = 4 * rows * (NH + 2 * NKV) * HS
    if kind == "attend":
        return {"bytes": qkv + 4 * rows * (NH * HS + NH), "flops": 4 * pairs * NH * HS}
    return {"bytes": 2 * qkv + 4 * rows * (2 * NH * HS + NH), "flops": 10 * pairs * NH * HS}


# ---- the same in 64 bits -------------------------------------------------------------

def _keep64(n, p, seed, step, site):
    """The kept elements, on the host in numpy: Philox4x32-10 with 64-bit products."""
    m32 = np.uint64(0xFFFFFFFF)
    ctr = np.zeros((4, (n + 3) // 4), np.uint64)
    ctr[0] = np.arange((n + 3) // 4, dtype=np.uint64)
    ctr[2], ctr[3] = step, 1 + site
    key = [seed & 0xFFFFFFFF, seed >> 32 & 0xFFFFFFFF]
    for r in range(10):
        lo, hi = np.uint64(0xD2511F53) * ctr[0], np.uint64(0xCD9E8D57) * ctr[2]
        ctr = np.stack(((hi >> np.uint64(32)) ^ ctr[1] ^ np.uint64((key[0] + r * 0x9E3779B9) & 0xFFFFFFFF), hi & m32,
                        (lo >> np.uint64(32)) ^ ctr[3] ^ np.uint64((key[1] + r * 0xBB67AE85) & 0xFFFFFFFF), lo & m32))
    return torch.from_numpy(ctr.T.reshape(-1)[:n] >= np.uint64(round(float(np.float32(p)) * 2 ** 32))).cuda()


def exact(case, seed):
    c, kind = case, case["kind"]
    s = prepare(case, seed)
    scale = 1.0 / (1.0 - float(np.float32(P_DROP)))
    if kind == "dropout":
        keep = _keep64(c["n"], P_DROP, s["seed"], STEP, SITE)
        return {"out": s["inp"].double() * keep * scale, "dinp": s["dout"].double() * keep * scale}
    if kind == "droplayer":
        rows, C = s["x"].shape
        f = (_keep64(rows * C, P_DROP, s["seed"], STEP, SITE).double() * scale).view(rows, C)
        res = s["x"].double() + s["y"].double() * f
        var, mean = torch.var_mean(res, 1, correction=0, keepdim=True)
        r, w, do = (var + 1e-5).rsqrt(), s["weight"].double(), s["dout"].double()
        n = (res - mean) * r
        back = (do * w * r).sub((do * w * r).sum(1, keepdim=True) / C).sub(n * ((do * w * n * r).sum(1, keepdim=True) / C))
        d = s["dres"].double() + back
        return {"res": res, "out": torch.addcmul(s["bias"].double(), n, w), "mean": mean.flatten(), "rstd": r.flatten(),
                "dinp": d, "dx": d, "dy": d * f, "dparam": torch.stack(((do * n).sum(0), do.sum(0)))}
    NH, NKV, HS = c["NH"], c["NKV"], c["HS"]
    G, scale, lens = NH // NKV, s["scale"], _lengths(c)
    out = torch.zeros_like(s["out"], dtype=torch.float64).view(-1, NH, HS)
    lse = torch.zeros_like(s["lse"], dtype=torch.float64)
    dqkv = torch.zeros_like(s["qkv"], dtype=torch.float64).view(-1, NH + 2 * NKV, HS) if kind == "backward" else None
    at = 0
    for b, n in enumerate(lens):
        if kind == "decode":
            q0, nq, k0 = b * c["Q"], c["Q"], b * c["cap"]
            rq, rk, rv = s["q"].view(-1, NH, HS), s["k"].view(-1, NKV, HS), s["v"].view(-1, NKV, HS)
        else:
            q0, nq, k0 = at, n, at
            rq = rk = rv = s["qkv"].view(-1, NH + 2 * NKV, HS)
            rk, rv = rk[:, NH:], rv[:, NH + NKV:]
        at += n
        late = torch.ones(nq, n, dtype=torch.bool, device="cuda").triu(n - nq + 1)
        for h in range(NH):
            q, k, v = rq[q0:q0 + nq, h].double(), rk[k0:k0 + n, h // G].double(), rv[k0:k0 + n, h // G].double()
            z = (q @ k.T * scale).masked_fill(late, -math.inf)
            if kind != "backward":
                lse[q0:q0 + nq, h] = torch.logsumexp(z, 1)
                out[q0:q0 + nq, h] = torch.exp(z - lse[q0:q0 + nq, h, None]) @ v
                continue
            p = torch.exp(z - s["lse"][q0:q0 + nq, h, None].double())
            do = s["dout"].view(-1, NH, HS)[q0:q0 + nq, h].double()
            dz = p * (do @ v.T - (do * s["out"].view(-1, NH, HS)[q0:q0 + nq, h].double()).sum(1, keepdim=True)) * scale
            dqkv[q0:q0 + nq, h] = dz @ k
            dqkv[k0:k0 + n, NH + h // G] += dz.T @ q
            dqkv[k0:k0 + n, NH + NKV + h // G] += p.T @ do
    if kind == "backward":
        return {"dqkv": dqkv.view_as(s["qkv"])}
    return {"out": out.view_as(s["out"]), "lse": lse}
