"""Generation from a cache in 8 bits as programs built on ugk have it, as cases to time and to check.

A case is a dict of plain values; its "kind" names what one pass is:

  step    the new rows of every sequence, which hold q, k and v side by side: k and v are stored in the cache
          behind what it holds, then the rows attend to it, causal. One row per sequence (the next token), a few
          (drafted tokens), or a prompt's. "weigh": the weight that each block of the cache got is added up, too
  store   prompts' keys and values stored in an empty cache, and read back
  evict   the blocks of least weight leave the tables
  verify  drafted tokens against the target's probabilities, from given random numbers. "sure": the drafts
          have no probabilities of their own

B sequences; HS is the size of a head, NH and NKV the numbers of query and key/value heads. The cache holds
blocks of 64 tokens in any order, whose numbers a table of "cap" tokens per sequence lists; "lens" says how full
it is: "equal" or "ragged" (lengths drawn from "len_seed"), and of "store" and of steps of more than eight rows also
how many rows are new. A block of a head holds whole numbers of up to 127 times a power of two.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

BLOCK = 64


def listed():
    return [
        # the next token of four sequences of the character-level model: a call of a few microseconds
        {"name": "step_text8", "kind": "step", "B": 4, "cap": 256, "Q": 1, "lens": "ragged", "len_seed": 2, "NH": 6, "NKV": 6,
         "HS": 64, "weigh": False},
        # the next token of 16 sequences of GPT-2-124M whose cache is to be kept short
        {"name": "step_gpt2", "kind": "step", "B": 16, "cap": 1024, "Q": 1, "lens": "ragged", "len_seed": 3, "NH": 12,
         "NKV": 12, "HS": 64, "weigh": True},
        # the next token of 24 long conversations, four query heads to a key/value head
        {"name": "step_long", "kind": "step", "B": 24, "cap": 16384, "Q": 1, "lens": "ragged", "len_seed": 4, "NH": 32,
         "NKV": 8, "HS": 128, "weigh": False},
        # four drafted tokens and the one before them, for each of 16 conversations
        {"name": "step_draft", "kind": "step", "B": 16, "cap": 8192, "Q": 5, "lens": "ragged", "len_seed": 5, "NH": 16,
         "NKV": 4, "HS": 128, "weigh": True},
        # prompts of up to 512 tokens behind long conversations
        {"name": "step_chunk", "kind": "step", "B": 4, "cap": 8192, "Q": 512, "lens": "ragged", "len_seed": 6, "NH": 16,
         "NKV": 4, "HS": 128, "weigh": False},
        # whole prompts of GPT-2-124M
        {"name": "step_prompt", "kind": "step", "B": 8, "cap": 1024, "Q": 1024, "lens": "equal", "len_seed": 0, "NH": 12,
         "NKV": 12, "HS": 64, "weigh": False},
        # GPT-2-124M's keys and values of a batch
        {"name": "store_gpt2", "kind": "store", "B": 8, "cap": 1024, "lens": "equal", "len_seed": 0, "NH": 12, "NKV": 12,
         "HS": 64},
        # documents of different lengths, heads of another size
        {"name": "store_odd", "kind": "store", "B": 13, "cap": 1500, "lens": "ragged", "len_seed": 7, "NH": 10, "NKV": 5,
         "HS": 80},
        # short caches of a small batch
        {"name": "evict_gpt2", "kind": "evict", "B": 16, "cap": 1024, "len_seed": 8, "keep": 8, "first": 1, "recent": 2},
        # the long ones of a server
        {"name": "evict_long", "kind": "evict", "B": 64, "cap": 262144, "len_seed": 9, "keep": 1024, "first": 1, "recent": 8},
        # drafts of the character-level model, looked up in the text so far
        {"name": "verify_text8", "kind": "verify", "B": 4, "K": 4, "V": 27, "sure": True},
        # drafts of GPT-2-124M's vocabulary
        {"name": "verify_gpt2", "kind": "verify", "B": 64, "K": 4, "V": 50257, "sure": False},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng, most):
    """(NH, NKV, HS): mostly heads of 64, now and then of 128, seldom of another size."""
    group = rng.choice((1, 1, 1, 2, 3, 4, 8))
    nkv = max(1, _log_int(rng, 1, most) // group)
    return nkv * group, nkv, rng.choice((64, 64, 64, 128, 128, 32, 80, 50))


def draw(rng):
    kind = rng.choice(("step", "step", "step", "step", "store", "evict", "verify", "verify"))
    seed, lens = rng.randrange(1000), rng.choice(("ragged", "ragged", "equal"))
    if kind == "evict":
        cap = _log_int(rng, 256, 262144)
        keep = _log_int(rng, 3, max(3, cap // BLOCK))
        first = rng.randrange(min(4, keep))
        return {"kind": kind, "B": _log_int(rng, 1, 64), "cap": cap, "len_seed": seed, "keep": keep, "first": first,
                "recent": rng.randrange(1, min(16, keep - first) + 1)}
    if kind == "verify":
        V, K = _log_int(rng, 27, 131072), rng.randrange(1, 9)
        return {"kind": kind, "B": _log_int(rng, 1, max(1, min(64, (1 << 25) // (V * K)))), "K": K, "V": V,
                "sure": rng.random() < 0.3}
    NH, NKV, HS = _heads(rng, 32)
    if kind == "store":
        cap = _log_int(rng, 16, 4096)
        B = _log_int(rng, 1, max(1, min(32, (1 << 22) // (cap * NKV * HS))))
        return {"kind": kind, "B": B, "cap": cap, "lens": lens, "len_seed": seed, "NH": NH, "NKV": NKV, "HS": HS}
    what = rng.choice(("next", "next", "draft", "prompt"))
    if what == "prompt":
        cap = _log_int(rng, 64, 8192)
        Q = _log_int(rng, 16, min(cap, 1024))
        B = _log_int(rng, 1, max(1, min(16, (1 << 27) // (cap * Q * NH), (1 << 23) // (cap * NKV * HS))))
    else:
        cap = _log_int(rng, 16, 16384)
        Q = 1 if what == "next" else rng.randrange(2, 9)
        B = _log_int(rng, 1, max(1, min(64, (1 << 27) // (cap * NKV * HS))))
    return {"kind": kind, "B": B, "cap": cap, "Q": Q, "lens": lens, "len_seed": seed, "NH": NH, "NKV": NKV, "HS": HS,
            "weigh": what != "prompt" and rng.random() < 0.4}


def _lengths(c):
    """(new rows, keys with them) of each sequence."""
    B, cap, kind = c["B"], c["cap"], c["kind"]
    rng = random.Random(c["len_seed"])
    if kind == "evict":
        return [(0, rng.randint(1, cap)) for _ in range(B)]
    most = cap if kind == "store" else c["Q"]
    if c["lens"] == "equal":
        return [(most, cap)] * B
    n = [rng.randint(1, most) if most > 8 else most for _ in range(B)]
    return [(x, x if kind == "store" else rng.randint(x, cap)) for x in n]


# ---- inputs ---------------------------------------------------------------------

def _rand(g, *shape, scale=1.0):
    t = torch.randn(*shape, generator=g, device="cuda")
    return t if scale == 1.0 else t.mul_(scale)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _place():
    """Where key i of a block stands in a row of the values' codes."""
    i = torch.arange(BLOCK, device="cuda")
    return i % 16 * 4 + i // 16


def _power(amax):
    """The scale of a block whose largest number is amax: the least power of two s with amax <= 127 s; 0 for 0."""
    m, x = torch.frexp(amax)
    e = (x - 7 + (m > 127 / 128).to(x.dtype)).clamp(-126, 121)
    return torch.where(amax > 0, ((e + 127) << 23).view(torch.float32), torch.zeros_like(amax))


def _codes(x, scale):
    return torch.round(x / torch.where(scale > 0, scale, torch.ones_like(scale))).clamp(-127, 127)


def _caches(g, blocks, NKV, HS, scale):
    """A cache that holds random rows."""
    HP = (HS + 15) // 16 * 16
    s = {}
    for name in ("k", "v"):
        x = _rand(g, blocks, NKV, BLOCK, HS, scale=scale)
        s[name + "s"] = _power(x.abs().amax((2, 3)))
        code = torch.zeros(blocks, NKV, BLOCK, HP, dtype=torch.int8, device="cuda")
        code[..., :HS] = _codes(x, s[name + "s"][:, :, None, None])
        s[name + "8"] = code
    at = torch.empty_like(s["v8"].transpose(2, 3), memory_format=torch.contiguous_format)
    at[..., _place()] = s["v8"].transpose(2, 3)
    s["v8"] = at
    return s


def prepare(case, seed):
    c, kind, B = case, case["kind"], case["B"]
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    if kind == "verify":
        K, V = c["K"], c["V"]
        rows = _rand(g, B, K + 1, V, scale=2.5)
        p = torch.softmax(rows, 2)
        q = torch.softmax(rows[:, :K] + _rand(g, B, K, V, scale=0.5), 2)  # a smaller model's, much like the target's
        draft = torch.multinomial(q.view(B * K, V), 1, generator=g).view(B, K).int()
        n = torch.randint(0, K + 1, (B,), generator=g, device="cuda") if B > 8 else torch.full((B,), K, device="cuda")
        e = lambda *s: torch.empty(*s, dtype=torch.int32, device="cuda")  # noqa: E731
        return {"case": c, "p": p, "q": None if c["sure"] else q, "draft": draft, "n_draft": n.int(),
                "u": torch.rand(B, K + 1, generator=g, device="cuda"), "accepted": e(B), "tokens": e(B, K + 1)}
    nb = (c["cap"] + BLOCK - 1) // BLOCK
    lens = _lengths(c)
    s = {"case": c, "k_len": _ints([n for _, n in lens]),
         "table": torch.randperm(B * nb, generator=g, device="cuda").int().view(B, nb)}
    if kind == "evict":
        # weights as attention leaves them: a few blocks have most, many have little, some none at all
        w = torch.exp(_rand(g, B, nb, scale=2.0)) * (torch.rand(B, nb, generator=g, device="cuda") > 0.1)
        i = torch.arange(nb, device="cuda")
        s["weight"] = w * (i < (s["k_len"][:, None] + BLOCK - 1) // BLOCK)
        s |= {"table_out": torch.empty_like(s["table"]), "len_out": torch.empty_like(s["k_len"]),
              "weight_out": torch.empty_like(w), "dropped": torch.empty_like(s["k_len"])}
        return s
    NH, NKV, HS = c["NH"], c["NKV"], c["HS"]
    start = [sum(n for n, _ in lens[:b]) for b in range(B + 1)]
    s["cu"] = _ints(start)
    s["max_q"] = max(n for n, _ in lens)
    s["qkv"] = _rand(g, start[-1], (NH + 2 * NKV) * HS)
    s |= _caches(g, B * nb, NKV, HS, 1.0)
    if kind == "store":
        s["k"], s["v"] = torch.empty(start[-1], NKV * HS, device="cuda"), torch.empty(start[-1], NKV * HS, device="cuda")
        return s
    s["scale"] = 1.0 / math.sqrt(HS)
    s["out"], s["lse"] = torch.empty(start[-1], NH * HS, device="cuda"), torch.empty(start[-1], NH, device="cuda")
    if c["weigh"]:
        s["before"] = torch.rand(B, nb, generator=g, device="cuda")
        s["weight"] = torch.empty(B, nb, device="cuda")
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


def _call(ugk, s, c):
    """The call's sequences, heads and row strides."""
    NH, NKV, HS = c["NH"], c["NKV"], c["HS"]
    ld = (NH + 2 * NKV) * HS
    return ugk.Cache8(nseq=c["B"], NH=NH, NKV=NKV, HS=HS, rows_q=s["qkv"].shape[0], max_q=s["max_q"], max_k=c["cap"],
                      nblocks=s["ks"].shape[0], causal=True, q_start=s["cu"][:-1], q_end=s["cu"][1:], k_len=s["k_len"],
                      table=s["table"], ldq=ld, ldk=ld, ldv=ld)


def _own_step(s, c):
    ugk = _ugk()
    NH, NKV, HS = c["NH"], c["NKV"], c["HS"]
    a, flat = _call(ugk, s, c), s["qkv"].view(-1)
    ugk.cache8_store(s["k8"], s["ks"], s["v8"], s["vs"], flat[NH * HS:], flat[(NH + NKV) * HS:], a)
    if not c["weigh"]:
        ugk.cache8_attention(s["out"], s["lse"], flat, s["k8"], s["ks"], s["v8"], s["vs"], a)
        return {k: s[k] for k in ("out", "lse", "ks", "vs")}
    s["weight"].copy_(s["before"])  # it accumulates
    ugk.cache8_attention(s["out"], s["lse"], flat, s["k8"], s["ks"], s["v8"], s["vs"], a, weight=s["weight"])
    return {k: s[k] for k in ("out", "lse", "ks", "vs", "weight")}


def _own_store(s, c):
    ugk = _ugk()
    NH, NKV, HS = c["NH"], c["NKV"], c["HS"]
    a, flat = _call(ugk, s, c), s["qkv"].view(-1)
    ugk.cache8_store(s["k8"], s["ks"], s["v8"], s["vs"], flat[NH * HS:], flat[(NH + NKV) * HS:], a)
    a.ldk = a.ldv = 0
    ugk.cache8_load(s["k"], s["v"], s["k8"], s["ks"], s["v8"], s["vs"], a)
    return {k: s[k] for k in ("k", "v", "ks", "vs")}


def _own_evict(s, c):
    _ugk().cache8_evict(s["table_out"], s["len_out"], s["weight_out"], s["dropped"], s["table"], s["k_len"], s["weight"],
                        c["B"], s["table"].shape[1], c["keep"], c["first"], c["recent"])
    return {k: s[k] for k in ("table_out", "len_out", "weight_out", "dropped")}


def _own_verify(s, c):
    _ugk().draft_verify(s["accepted"], s["tokens"], s["p"], s["q"], s["draft"], s["n_draft"], s["u"], c["B"], c["K"], c["V"])
    return {"accepted": s["accepted"], "tokens": s["tokens"]}


_OWN = {"step": _own_step, "store": _own_store, "evict": _own_evict, "verify": _own_verify}


def _rows(s):
    """The sequence of each row and its place in it."""
    r = torch.arange(s["qkv"].shape[0], device="cuda")
    b = torch.searchsorted(s["cu"][1:], r, right=True)
    return b, r - s["cu"].long()[b]


def _three(s, c):
    """q, k and v as (rows, heads, HS)."""
    NH, NKV, HS = c["NH"], c["NKV"], c["HS"]
    t = s["qkv"].view(-1, NH + 2 * NKV, HS)
    return t[:, :NH], t[:, NH:NH + NKV], t[:, NH + NKV:]


def _put(s, c, x, code, scale, values):
    """Rows x (rows, NKV, HS) into the codes: block by block, all that a sequence touches at once."""
    HS, nt = c["HS"], (s["max_q"] + 2 * BLOCK - 2) // BLOCK
    start, end = s["cu"][:-1].long(), s["k_len"].long()
    begin = end - (s["cu"][1:].long() - start)
    # a sequence that touches fewer than nt blocks has its last one several times, with the same content
    j = torch.minimum(begin[:, None] // BLOCK + torch.arange(nt, device="cuda"), (end[:, None] - 1) // BLOCK)
    block = s["table"].long().gather(1, j)
    pos = j[:, :, None] * BLOCK + torch.arange(BLOCK, device="cuda")
    old = pos < begin[:, None, None]
    new = ~old & (pos < end[:, None, None])
    row = torch.where(new, start[:, None, None] + pos - begin[:, None, None], 0)
    rows = torch.where(new[..., None, None], x[row], 0.0).permute(0, 1, 3, 2, 4)  # (B, nt, NKV, 64, HS)
    need = _power(rows.abs().amax((3, 4)))
    had = torch.where(old[:, :, :1], scale[block], 0.0)
    now = torch.maximum(need, had)
    kept = code[block]
    if values:
        kept = kept[..., _place()].transpose(3, 4)
    kept = kept[..., :HS].float()
    again = _codes(kept * had[..., None, None], now[..., None, None])
    is_new, is_old = new[:, :, None, :, None], old[:, :, None, :, None]
    out = torch.where(is_new, _codes(rows, now[..., None, None]), torch.where(is_old, again, kept))
    whole = torch.zeros(*out.shape[:4], code.shape[2 if values else 3], dtype=torch.int8, device="cuda")
    whole[..., :HS] = out
    if values:
        at = torch.empty_like(whole.transpose(3, 4), memory_format=torch.contiguous_format)
        at[..., _place()] = whole.transpose(3, 4)
        whole = at
    code[block] = whole
    scale[block] = now


def _take(s, c, code, scale, values):
    """The numbers that the codes stand for, (B, NKV, keys, HS)."""
    block = s["table"].long()
    t = code[block]
    if values:
        t = t[..., _place()].transpose(3, 4)
    t = t[..., :c["HS"]].float() * scale[block][..., None, None]
    B, nb, NKV = t.shape[:3]
    return t.permute(0, 2, 1, 3, 4).reshape(B, NKV, nb * BLOCK, c["HS"])


def _plain_step(s, c):
    NH, NKV, HS, B = c["NH"], c["NKV"], c["HS"], c["B"]
    q, k, v = _three(s, c)
    _put(s, c, k, s["k8"], s["ks"], False)
    _put(s, c, v, s["v8"], s["vs"], True)
    K, V = _take(s, c, s["k8"], s["ks"], False), _take(s, c, s["v8"], s["vs"], True)
    start, end, lk = s["cu"][:-1].long()[:, None], s["cu"][1:].long()[:, None], s["k_len"].long()[:, None]
    i, j = torch.arange(s["max_q"], device="cuda"), torch.arange(K.shape[2], device="cuda")
    in_q = i < end - start
    at = torch.where(in_q, start + i, 0)
    Q = q[at].view(B, -1, NKV, NH // NKV, HS).permute(0, 2, 3, 1, 4).reshape(B, NKV, -1, HS)
    S = torch.matmul(Q, K.transpose(2, 3)).view(B, NKV, NH // NKV, -1, K.shape[2]).mul_(s["scale"])
    ok = in_q[:, :, None] & (j <= i[:, None] + (lk - (end - start))[:, :, None])
    S.masked_fill_(~ok[:, None, None], float("-inf"))
    m = S.amax(4, keepdim=True)
    m = torch.where(m == float("-inf"), 0.0, m)
    P = S.sub_(m).exp_()
    l = P.sum(4, keepdim=True)
    inv = 1.0 / torch.where(l == 0, 1.0, l)
    V = torch.where((j < lk)[:, None, :, None], V, 0.0)  # what lies behind a sequence is no number of it
    O = torch.matmul(P.view(B, NKV, -1, K.shape[2]), V).view(B, NKV, NH // NKV, -1, HS) * inv
    lse = (m + torch.log(l)).squeeze(4)
    b, row = _rows(s)
    r = {"out": O.permute(0, 3, 1, 2, 4)[b, row].flatten(1), "lse": lse.permute(0, 3, 1, 2)[b, row].flatten(1),
         "ks": s["ks"], "vs": s["vs"]}
    if c["weigh"]:
        r["weight"] = s["before"] + P.mul_(inv).sum((1, 2, 3)).view(B, -1, BLOCK).sum(2)
    return r


def _plain_store(s, c):
    _, k, v = _three(s, c)
    _put(s, c, k, s["k8"], s["ks"], False)
    _put(s, c, v, s["v8"], s["vs"], True)
    b, row = _rows(s)
    K, V = (_take(s, c, s[n + "8"], s[n + "s"], n == "v").transpose(1, 2)[b, row].flatten(1) for n in ("k", "v"))
    return {"k": K, "v": V, "ks": s["ks"], "vs": s["vs"]}


def _plain_evict(s, c):
    table, weight, keep, first, recent = s["table"], s["weight"], c["keep"], c["first"], c["recent"]
    nb = table.shape[1]
    n = (s["k_len"].long() + BLOCK - 1) // BLOCK
    i = torch.arange(nb, device="cuda")
    drop = (n - keep).clamp(min=0)
    may = (i >= first) & (i < (n - recent)[:, None])
    order = torch.sort(torch.where(may, weight, float("inf")), dim=1, stable=True).indices
    rank = torch.empty_like(order).scatter_(1, order, i.expand_as(order).contiguous())
    gone = rank < drop[:, None]
    order = torch.sort(gone.int(), dim=1, stable=True).indices  # those that stay, in order, then those that go
    left = i < (n - drop)[:, None]
    return {"table_out": table.gather(1, order), "len_out": (s["k_len"] - drop * BLOCK).int(),
            "weight_out": torch.where(left, weight.gather(1, order), 0.0), "dropped": drop.int()}


def _plain_verify(s, c):
    B, K, V = c["B"], c["K"], c["V"]
    p, q, draft, n, u = s["p"], s["q"], s["draft"].long(), s["n_draft"].long(), s["u"].double()
    i = torch.arange(K, device="cuda")
    pt = p[:, :K].gather(2, draft[..., None]).squeeze(2).double()
    qt = torch.ones_like(pt) if q is None else q.gather(2, draft[..., None]).squeeze(2).double()
    ok = (u[:, :K] * qt < pt) & (i < n[:, None])
    a = ok.long().cumprod(1).sum(1)
    row = p.gather(1, a[:, None, None].expand(B, 1, V)).squeeze(1).double()
    at = a.clamp(max=K - 1)
    if q is None:
        less = torch.zeros_like(row).scatter_(1, draft.gather(1, at[:, None]), 2.0)
    else:
        less = q.gather(1, at[:, None, None].expand(B, 1, V)).squeeze(1).double()
    rest = torch.where((a < n)[:, None], (row - less).clamp(min=0), row)
    rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, row)
    sums = rest.cumsum(1)
    token = (sums <= u[:, K:] * sums[:, -1:]).sum(1).clamp(max=V - 1)
    i = torch.arange(K + 1, device="cuda")
    longer = torch.cat((draft, draft[:, :1]), 1)
    tokens = torch.where(i < a[:, None], longer, torch.where(i == a[:, None], token[:, None], -1))
    return {"accepted": a.int(), "tokens": tokens.int()}


_PLAIN = {"step": _plain_step, "store": _plain_store, "evict": _plain_evict, "verify": _plain_verify}


# ---- what a pass cannot do without -------------------------------------------------

def work(case):
    """Bytes with each input read once and each output written once, and the float operations."""
    c, kind, B = case, case["kind"], case["B"]
    if kind == "verify":  # a row of the target's probabilities, and of the drafts', per sequence
        return {"bytes": 4 * B * (c["V"] * (1 if c["sure"] else 2) + 3 * c["K"] + 3), "flops": 3 * B * c["V"]}
    lens = _lengths(c)
    blocks = sum((n + BLOCK - 1) // BLOCK for _, n in lens)
    if kind == "evict":  # table and weight read and written
        return {"bytes": 16 * B * ((c["cap"] + BLOCK - 1) // BLOCK) + 12 * B, "flops": blocks}
    NH, NKV, HS = c["NH"], c["NKV"], c["HS"]
    new, keys = sum(n for n, _ in lens), sum(n for _, n in lens)
    if kind == "store":  # rows read, codes written; codes read, rows written
        return {"bytes": 2 * new * NKV * HS * 10 + 16 * blocks * NKV, "flops": 4 * new * NKV * HS}
    pairs = sum(q * n - q * (q - 1) // 2 for q, n in lens)
    # new rows read, their codes written, all codes read, out and lse written
    return {"bytes": 4 * new * (NH + 2 * NKV) * HS + 2 * (new + keys) * NKV * HS + 8 * blocks * NKV + 4 * new * (NH * HS + NH) +
            (8 * blocks if c["weigh"] else 0), "flops": 4 * pairs * NH * HS}


# ---- the same in 64 bits -------------------------------------------------------------

def _scale64(top):
    """The least power of two s, 2^-126 to 2^121, with top <= 127 s, in numpy; 0 for 0."""
    e = np.clip(np.ceil(np.log2(np.maximum(top, 1e-300) / 127)), -126, 121)
    e = np.where(top > 127 * np.exp2(e), e + 1, np.where(top <= 127 * np.exp2(e - 1), e - 1, e)).clip(-126, 121)
    return np.where(top > 0, np.exp2(e), 0.0)


def _after(s, c, name, x, lens):
    """What the cache holds once rows x are stored: (scales of all blocks, per sequence its keys (n, NKV, HS))."""
    HS, table = c["HS"], s["table"].cpu().numpy()
    scales = s[name + "s"].double().cpu().numpy()
    code = s[name + "8"]
    order = torch.tensor([(i % 16) * 4 + i // 16 for i in range(BLOCK)], device="cuda")
    held, at = [], 0
    for b, (n, end) in enumerate(lens):
        begin, nb = end - n, (end + BLOCK - 1) // BLOCK
        t = code[torch.from_numpy(table[b, :nb]).long().cuda()]
        t = t[:, :, :HS, order].permute(0, 3, 1, 2) if name == "v" else t[..., :HS].permute(0, 2, 1, 3)
        t = (t.double() * torch.from_numpy(scales[table[b, :nb]]).cuda()[:, None, :, None]).flatten(0, 1)[:end].clone()
        new = x[at:at + n].double()
        at += n
        for j in range(begin // BLOCK, nb):
            lo, hi, mid = j * BLOCK, min(end, (j + 1) * BLOCK), max(begin, j * BLOCK)
            rows = new[mid - begin:hi - begin]
            sc = _scale64(rows.abs().amax((0, 2)).cpu().numpy())
            if mid > lo:
                sc = np.maximum(sc, scales[table[b, j]])
            scales[table[b, j]] = sc
            w = torch.from_numpy(np.where(sc > 0, sc, 1.0)).cuda()[None, :, None]
            t[lo:mid] = torch.clamp((t[lo:mid] / w).round(), -127, 127) * w
            t[mid:hi] = torch.clamp((rows / w).round(), -127, 127) * w
        held.append(t)
    return torch.from_numpy(scales).cuda(), held


def exact(case, seed):
    c, kind, B = case, case["kind"], case["B"]
    s = prepare(case, seed)
    if kind == "verify":
        return _exact_verify(s, c)
    lens = _lengths(c)
    if kind == "evict":
        return _exact_evict(s, c, lens)
    NH, NKV, HS = c["NH"], c["NKV"], c["HS"]
    rows = s["qkv"].view(-1, NH + 2 * NKV, HS)
    ks, held_k = _after(s, c, "k", rows[:, NH:NH + NKV], lens)
    vs, held_v = _after(s, c, "v", rows[:, NH + NKV:], lens)
    r = {"ks": ks, "vs": vs}
    if kind == "store":
        return r | {"k": torch.cat(held_k).flatten(1), "v": torch.cat(held_v).flatten(1)}
    out = torch.zeros(len(rows), NH, HS, dtype=torch.float64, device="cuda")
    lse = torch.zeros(len(rows), NH, dtype=torch.float64, device="cuda")
    weight = s["before"].double() if c["weigh"] else None
    at = 0
    for b, (n, end) in enumerate(lens):
        late = torch.ones(n, end, dtype=torch.bool, device="cuda").triu(end - n + 1)
        for h in range(NH):
            k, v = held_k[b][:, h // (NH // NKV)], held_v[b][:, h // (NH // NKV)]
            z = (rows[at:at + n, h].double() @ k.T / math.sqrt(HS)).masked_fill(late, -math.inf)
            lse[at:at + n, h] = torch.logsumexp(z, 1)
            p = torch.exp(z - lse[at:at + n, h, None])
            out[at:at + n, h] = p @ v
            if weight is not None:
                got = p.sum(0)
                nb = (end + BLOCK - 1) // BLOCK
                weight[b, :nb] += torch.nn.functional.pad(got, (0, nb * BLOCK - end)).view(nb, BLOCK).sum(1)
        at += n
    return r | {"out": out.flatten(1), "lse": lse} | ({} if weight is None else {"weight": weight})


def _exact_evict(s, c, lens):
    table, weight = s["table"].cpu().numpy(), s["weight"].cpu().numpy()
    t, w, ln, dropped = table.copy(), np.zeros_like(weight), [], []
    for b, (_, end) in enumerate(lens):
        n = -(-end // BLOCK)
        d = max(0, n - c["keep"])
        may = sorted(range(c["first"], n - c["recent"]), key=lambda i: (weight[b, i], i))
        gone = set(may[:d])
        stay = [i for i in range(n) if i not in gone]
        t[b] = table[b, stay + list(range(n, table.shape[1])) + sorted(gone)]
        w[b, :len(stay)] = weight[b, stay]
        ln.append(end - BLOCK * d)
        dropped.append(d)
    return {"table_out": torch.from_numpy(t).cuda(), "len_out": _ints(ln), "weight_out": torch.from_numpy(w).double().cuda(),
            "dropped": _ints(dropped)}


def _exact_verify(s, c):
    K = c["K"]
    draft, n, u = s["draft"].cpu().numpy(), s["n_draft"].cpu().numpy(), s["u"].double().cpu().numpy()
    accepted, tokens = [], np.full((c["B"], K + 1), -1, np.int32)
    for b in range(c["B"]):
        i = 0
        while i < n[b]:
            t = int(draft[b, i])
            if not u[b, i] * (1.0 if s["q"] is None else float(s["q"][b, i, t])) < float(s["p"][b, i, t]):
                break
            tokens[b, i] = t
            i += 1
        rest = s["p"][b, i].double().cpu().numpy()
        if i < n[b]:
            less = np.eye(1, c["V"], draft[b, i])[0] if s["q"] is None else s["q"][b, i].double().cpu().numpy()
            r = np.maximum(rest - less, 0.0) if s["q"] is not None else rest * (1.0 - less)
            rest = r if r.sum() > 0 else rest
        sums = np.cumsum(rest)
        tokens[b, i] = min(int(np.searchsorted(sums, u[b, K] * sums[-1], side="right")), c["V"] - 1)
        accepted.append(i)
    return {"accepted": _ints(accepted), "tokens": torch.from_numpy(tokens).cuda()}
