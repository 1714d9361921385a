"""The operators of a guarded serving path over an 8-bit paged cache, as cases to time and compare.

rope     rotary positions of a projection's heads (far positions, a part of the head, both pair layouts), and the
         gradient in training
append   a step's keys and values rotated, quantized and written to a paged cache, the queries rotated beside them
attend   attention of a step's queries over the cache: one token a sequence, chunks of a prompt, or both in one batch
step     one layer's decode step: append, then attend

A cache is (pages, kv heads, slots of a page, 2 head size): keys, then values, in e4m3 or int8 codes; scales is
(pages, kv heads, 2) fp32, for the page's keys and its values.  Sequence r has query tokens start[r] .. start[r + 1],
the last of its length[r] positions; position p is in page table[r, p // slots], slot p % slots.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CODES = {"e4m3": (torch.float8_e4m3fn, 448.0, 0.875, 9), "int8": (torch.int8, 127.0, 127.0 / 128.0, 7)}


# ---------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # The smallest rotation: the query heads of 16 sequences at a decode step of a long-context service, positions
        # scaled by 4; bound by latency.
        {"name": "rope_decode_16", "kind": "rope", "tokens": 16, "heads": 32, "dim": 128, "rot": 128, "dtype": "bf16",
         "interleaved": False, "far": 131072, "factor": 4.0, "backward": False},
        # A training step's rotation and its gradient: 8192 tokens of 32 heads.
        {"name": "rope_train_8192", "kind": "rope", "tokens": 8192, "heads": 32, "dim": 128, "rot": 128,
         "dtype": "bf16", "interleaved": False, "far": 8192, "factor": 1.0, "backward": True},
        # A prompt of odd length of a model that rotates adjacent pairs in a part of each head, in fp16.
        {"name": "rope_part_4099", "kind": "rope", "tokens": 4099, "heads": 12, "dim": 80, "rot": 48, "dtype": "fp16",
         "interleaved": True, "far": 1000003, "factor": 8.0, "backward": False},
        # The append of a decode step: 64 sequences of 512-2048 tokens, 16 query and 8 key heads of 128, pages of 16.
        {"name": "append_decode_64", "kind": "append", "seqs": 64, "lo": 512, "hi": 2048, "chunks": 0, "chunk": 1,
         "heads": 16, "kv_heads": 8, "dim": 128, "rot": 128, "page": 16, "cache": "e4m3", "dtype": "bf16",
         "interleaved": False, "window": 0, "lens": 1},
        # The append of a prefill step: four prompt chunks of about 4096 tokens, 32 query and 8 key heads.
        {"name": "append_prefill_16k", "kind": "append", "seqs": 4, "lo": 4096, "hi": 8192, "chunks": 4, "chunk": 4096,
         "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "page": 16, "cache": "e4m3", "dtype": "bf16",
         "interleaved": False, "window": 0, "lens": 2},
        # A mixed step (one chunk of 500 tokens beside 40 decoding sequences) into an int8 cache, half of each head of
        # 64 rotated in adjacent pairs, pages of 32.
        {"name": "append_mixed_int8", "kind": "append", "seqs": 41, "lo": 100, "hi": 4000, "chunks": 1, "chunk": 500,
         "heads": 12, "kv_heads": 12, "dim": 64, "rot": 32, "page": 32, "cache": "int8", "dtype": "fp16",
         "interleaved": True, "window": 0, "lens": 3},
        # One sequence of about 500 tokens, one new token: the smallest attention, bound by latency.
        {"name": "attend_decode_1", "kind": "attend", "seqs": 1, "lo": 490, "hi": 510, "chunks": 0, "chunk": 1,
         "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "page": 16, "cache": "int8", "dtype": "bf16",
         "interleaved": False, "window": 0, "lens": 4},
        # The decode step of 64 sequences of 512-2048 tokens.
        {"name": "attend_decode_64", "kind": "attend", "seqs": 64, "lo": 512, "hi": 2048, "chunks": 0, "chunk": 1,
         "heads": 16, "kv_heads": 8, "dim": 128, "rot": 128, "page": 16, "cache": "e4m3", "dtype": "bf16",
         "interleaved": False, "window": 0, "lens": 5},
        # Four long conversations of 100 000 to 131 072 tokens, one new token each.
        {"name": "attend_decode_long", "kind": "attend", "seqs": 4, "lo": 100000, "hi": 131072, "chunks": 0,
         "chunk": 1, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "page": 16, "cache": "e4m3",
         "dtype": "bf16", "interleaved": False, "window": 0, "lens": 6},
        # A prefill step: two prompt chunks of 2048 tokens behind contexts of up to 6000.
        {"name": "attend_prefill_4096", "kind": "attend", "seqs": 2, "lo": 4096, "hi": 8192, "chunks": 2,
         "chunk": 2048, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "page": 16, "cache": "e4m3",
         "dtype": "bf16", "interleaved": False, "window": 0, "lens": 7},
        # A mixed step under a sliding window of 1024: one chunk of 500 tokens beside 23 decoding sequences, heads of
        # 64, int8, fp16, pages of 32.
        {"name": "attend_mixed_window", "kind": "attend", "seqs": 24, "lo": 600, "hi": 4000, "chunks": 1, "chunk": 500,
         "heads": 24, "kv_heads": 4, "dim": 64, "rot": 64, "page": 32, "cache": "int8", "dtype": "fp16",
         "interleaved": False, "window": 1024, "lens": 8},
        # One layer's decode step, append and attention together: 32 sequences of 1000 to 4000 tokens.
        {"name": "step_decode_32", "kind": "step", "seqs": 32, "lo": 1000, "hi": 4000, "chunks": 0, "chunk": 1,
         "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "page": 16, "cache": "e4m3", "dtype": "bf16",
         "interleaved": False, "window": 0, "lens": 9},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.25:
        dim = rng.choice([48, 64, 80, 96, 128, 256])
        heads = rng.choice([1, 4, 12, 16, 32])
        rot = min(dim, rng.choice([16, 32, 48, dim, dim]))
        back = rng.random() < 0.5
        most = 8192 * 32 * 128 // (heads * dim)
        return {"kind": "rope", "tokens": min(_log(rng, 1, 16384), most), "heads": heads, "dim": dim, "rot": rot,
                "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "interleaved": rng.random() < 0.5,
                "far": _log(rng, 100000, 1000000), "factor": rng.choice([1.0, 2.0, 4.0, 8.0]), "backward": back}
    kind = rng.choice(["append", "attend", "attend", "step"])
    kv_heads = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 7, 8, 16])
    dim = rng.choice([64, 80, 96, 128, 128, 256])
    seqs = _log(rng, 1, 128)
    most = min(131072, 4 * 131072 * 8 * 128 // (seqs * kv_heads * dim * 2))     # no more cache than the longest case
    hi = _log(rng, 40, min(most, 65536 // max(1, seqs // 4)))
    chunks = 0 if rng.random() < 0.5 else rng.randint(1, min(seqs, 4))
    work = 2 * 2048 * 6144 * 32 * 128                                           # no more scores than the prefill case
    chunk = 1 if not chunks else max(2, min(_log(rng, 2, 2048), hi, work // (seqs * hi * kv_heads * group * dim)))
    return {"kind": kind, "seqs": seqs, "lo": max(1, hi // 4), "hi": hi, "chunks": chunks, "chunk": chunk,
            "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "rot": rng.choice([dim, dim, 32]),
            "page": rng.choice([8, 16, 16, 32, 64]), "cache": rng.choice(["e4m3", "e4m3", "int8"]),
            "dtype": rng.choice(["bf16", "bf16", "fp16"]), "interleaved": rng.random() < 0.3,
            "window": rng.choice([0, 0, 0, 128, 1000]), "lens": rng.randrange(1 << 20)}


# --------------------------------------------------------------------------------------------------- the inputs
def _lengths(case):
    """(lengths, query lengths) of the step's sequences: spread over their range, the first ones with a chunk."""
    rng = random.Random(case["lens"])
    length = [_log(rng, case["lo"], case["hi"]) for _ in range(case["seqs"])]
    new = [1] * case["seqs"]
    for i in range(case["chunks"]):
        new[i] = max(1, case["chunk"] - rng.randrange(max(1, case["chunk"] // 8)))
        length[i] = max(length[i], new[i])
    return length, new


def _randn(shape, gen):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rot = case["rot"]
    i = torch.arange(rot // 2, device="cuda", dtype=torch.float64)
    factor = case.get("factor", 1.0)
    # what a rotation by position keeps per model: the turns a pair makes per position, and the factor on the result
    turns = 500000.0 ** (-2.0 * i / rot) / (2.0 * math.pi) / factor
    state = {"case": case, "turns": turns, "mscale": 1.0 + 0.1 * math.log(factor)}
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "rope":
        T, H, D = case["tokens"], case["heads"], case["dim"]
        # the heads are a part of a fused projection's output: rows are further apart than the heads are wide
        wide = _randn((T, (H + 2) * D), gen).to(dtype)
        x = wide[:, :H * D].view(T, H, D)
        if case["far"] > T and case["tokens"] < 1024:                            # each row a sequence of its own
            pos = torch.randint(0, case["far"], (T,), generator=gen, device="cuda")
        else:                                                                    # one run of a sequence
            pos = torch.arange(T, device="cuda") + (case["far"] - T if case["far"] > T else 0)
        state |= {"x": x, "positions": pos}
        if case["backward"]:
            x.requires_grad_(True)
            state["dy"] = _randn((T, H, D), gen).to(dtype)
        return state

    length, new = _lengths(case)
    N, D, Hq, Hk = case["page"], case["dim"], case["heads"], case["kv_heads"]
    R, T, W = len(length), sum(new), -(-max(length) // N)
    used = [-(-n // N) for n in length]
    NB = sum(used) + 3
    perm = torch.randperm(NB, generator=gen, device="cuda").to(torch.int32)
    first = torch.tensor([0] + used, device="cuda").cumsum(0)[:-1]
    at = first[:, None] + torch.arange(W, device="cuda")
    live = torch.arange(W, device="cuda") < torch.tensor(used, device="cuda")[:, None]
    table = torch.where(live, perm[at.clamp(max=NB - 1)], torch.zeros_like(perm[:1]))
    # what earlier steps left in the cache: a quantized page is its largest value at the code's largest
    codes_t, top, _, _ = CODES[case["cache"]]
    kv = torch.empty(NB, Hk, N, 2 * D, dtype=torch.uint8, device="cuda")
    scales = torch.empty(NB, Hk, 2, device="cuda")
    exact_scales = case["kind"] != "attend"          # pages that this append wrote have powers of two
    for b in range(0, NB, 4096):                     # (a few large pieces, to bound the fp32 copy)
        e = min(NB, b + 4096)
        x = _randn((e - b, Hk, N, 2, D), gen) * (0.3 + 1.7 * torch.rand(1, Hk, 1, 2, D, generator=gen, device="cuda"))
        sc = x.abs().amax((2, 4)) / top
        if exact_scales:
            sc = torch.exp2(torch.ceil(torch.log2(sc)))
        y = x / sc[:, :, None, :, None]
        y = (y.round() if codes_t is torch.int8 else y).to(codes_t).view(torch.uint8)
        kv[b:e] = y.reshape(e - b, Hk, N, 2 * D)
        scales[b:e] = sc
    start = torch.tensor([0] + new, device="cuda").cumsum(0).to(torch.int32)
    qkv = _randn((T, (Hq + 2 * Hk) * D), gen).to(dtype)
    q, k, v = (t.view(T, -1, D) for t in qkv.split([Hq * D, Hk * D, Hk * D], 1))
    state |= {"q": q, "k": k, "v": v, "kv": kv.view(codes_t), "scales": scales, "start": start, "table": table,
              "length": torch.tensor(length, device="cuda", dtype=torch.int32), "most": max(new)}
    return state


# ---------------------------------------------------------------------------------------------- the plain forms
def _angles(turns, mscale, positions):
    t = positions.double()[:, None] * turns
    a = (t - t.round()) * (2.0 * math.pi)
    return (torch.cos(a) * mscale).float()[:, None], (torch.sin(a) * mscale).float()[:, None]


def _turned(x, c, s, rot, interleaved):
    y = x.clone()
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    if interleaved:
        y[..., 0:rot:2], y[..., 1:rot:2] = a * c - b * s, b * c + a * s
    else:
        y[..., :rot // 2], y[..., rot // 2:rot] = a * c - b * s, b * c + a * s
    return y


def _plain_rope(s):
    case, x = s["case"], s["x"]
    rot, inter = case["rot"], case["interleaved"]
    c, sn = _angles(s["turns"], s["mscale"], s["positions"])
    y = _turned(x.detach().float(), c, sn, rot, inter).to(x.dtype)
    if not case["backward"]:
        return y
    return {"y": y, "dx": _turned(s["dy"].float(), c, -sn, rot, inter).to(x.dtype)}


def _rows(s, T):
    """Each token's sequence and position."""
    t = torch.arange(T, device="cuda", dtype=torch.int32)
    r = torch.searchsorted(s["start"][1:].contiguous(), t, right=True)
    n = s["start"][r + 1] - s["start"][r]
    return r, (s["length"][r] - n + (t - s["start"][r])).long()


def _power(amax, m_top, e_top):
    """The smallest power of two whose product with the largest code holds amax."""
    m, e = torch.frexp(amax)
    e = torch.where(amax == 0, torch.full_like(e, -126), e - e_top + (m > m_top))
    return torch.ldexp(torch.ones_like(amax), e.clamp(-126, 120))


def _round(x, codes_t, top):
    if codes_t is torch.int8:
        return x.round().clamp(-top, top).to(torch.int8).view(torch.uint8)
    return x.to(codes_t).view(torch.uint8)


def _plain_append(s):
    case, kv, scales = s["case"], s["kv"], s["scales"]
    codes_t, top, m_top, e_top = CODES[case["cache"]]
    N, D, T = case["page"], case["dim"], s["k"].shape[0]
    r, pos = _rows(s, T)
    c, sn = _angles(s["turns"], s["mscale"], pos)
    q = _turned(s["q"].float(), c, sn, case["rot"], case["interleaved"]).to(s["q"].dtype)
    x = torch.stack([_turned(s["k"].float(), c, sn, case["rot"], case["interleaved"]), s["v"].float()], 2)
    page, slot = s["table"][r, pos // N].long(), pos % N
    NB, Hk = scales.shape[:2]
    amax = torch.zeros_like(scales).index_reduce_(0, page, x.abs().amax(-1), "amax")
    anew = torch.zeros(NB, device="cuda").index_reduce_(0, page, (slot == 0).float(), "amax") > 0
    touched = torch.zeros(NB, device="cuda").index_fill_(0, page, 1.0) > 0
    need = _power(amax, m_top, e_top)
    now = torch.where(anew[:, None, None], need, torch.maximum(scales, need))
    now = torch.where(touched[:, None, None], now, scales)
    # the codes already in the pages of this call, at the pages' new scales
    ratio = (scales / now)[page][:, :, None, :, None]
    raw = kv.view(torch.uint8)
    old = raw[page].view(codes_t).float().view(T, Hk, N, 2, D)
    moved = _round(old * ratio, codes_t, top).view(T, Hk, N, 2 * D)
    keep = (anew[page][:, None, None, None, None] | (ratio == 1)).expand(T, Hk, 1, 2, D).reshape(T, Hk, 1, 2 * D)
    raw[page] = torch.where(keep, raw[page], moved)
    raw[page, :, slot] = _round(x / now[page][..., None], codes_t, top).view(T, Hk, 2 * D)
    scales.copy_(now)
    return {"q": q, "kv": kv, "scales": scales}


def _plain_attend(s, q):
    case, kv, scales = s["case"], s["kv"], s["scales"]
    N, D, Hq, Hk = case["page"], case["dim"], case["heads"], case["kv_heads"]
    g, T, Q = Hq // Hk, q.shape[0], s["most"]
    R, W = s["table"].shape
    page = s["table"].long()
    x = kv.view(torch.uint8)[page].view(kv.dtype).float().view(R, W, Hk, N, 2, D) * scales[page][:, :, :, None, :, None]
    k = x[..., 0, :].transpose(1, 2).reshape(R, Hk, W * N, D)
    v = x[..., 1, :].transpose(1, 2).reshape(R, Hk, W * N, D)
    del x
    n = (s["start"][1:] - s["start"][:-1]).long()
    i = torch.arange(Q, device="cuda")
    rows = (s["start"][:-1, None] + i).clamp(max=T - 1).long()
    qq = q.float()[rows].view(R, Q, Hk, g, D).permute(0, 2, 3, 1, 4).reshape(R, Hk, g * Q, D)
    pos = (s["length"].long() - n)[:, None] + i
    key = torch.arange(W * N, device="cuda")
    seen = (key <= pos[..., None]) & (i < n[:, None])[..., None]
    if case["window"]:
        seen &= key > pos[..., None] - case["window"]
    p = torch.matmul(qq, k.transpose(2, 3)).view(R, Hk, g, Q, W * N) * D ** -0.5
    p = torch.where(seen[:, None, None], p, torch.full((), -math.inf, device="cuda"))
    m = p.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = torch.exp(p - m)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(R, Hk, g * Q, W * N), v).view(R, Hk, g, Q, D) / torch.where(total == 0, 1.0, total)
    r, _ = _rows(s, T)
    at = torch.arange(T, device="cuda") - s["start"][r].long()
    lse = (m + torch.log(total))[..., 0]
    return {"o": o[r, :, :, at].reshape(T, Hq, D).to(q.dtype), "lse": lse[r, :, :, at].reshape(T, Hq)}


# ------------------------------------------------------------------------------------------------ the operators
def _own_rope(s):
    from sdcguard_amd import rope
    case, x = s["case"], s["x"]
    y = rope.rotate(x, s["positions"], s["turns"], interleaved=case["interleaved"], mscale=s["mscale"])
    if not case["backward"]:
        return y
    return {"y": y.detach(), "dx": torch.autograd.grad(y, x, s["dy"])[0]}


def _own_append(s):
    from sdcguard_amd import kv_attn
    case = s["case"]
    q = kv_attn.kv_append(s["k"], s["v"], s["kv"], s["scales"], s["start"], s["length"], s["table"], turns=s["turns"],
                          interleaved=case["interleaved"], mscale=s["mscale"], query=s["q"])
    return {"q": q, "kv": s["kv"], "scales": s["scales"]}


def _own_attend(s, q):
    from sdcguard_amd import kv_attn
    case = s["case"]
    o, lse = kv_attn.kv_attend(q, s["kv"], s["scales"], s["start"], s["length"], s["table"], window=case["window"],
                               return_lse=True)
    return {"o": o, "lse": lse}


def run(state):
    kind = state["case"]["kind"]
    if kind == "rope":
        return _own_rope(state) if own else _plain_rope(state)
    append, attend = (_own_append, _own_attend) if own else (_plain_append, _plain_attend)
    if kind == "append":
        return append(state)
    if kind == "attend":
        return attend(state, state["q"])
    done = append(state)
    return {**done, **attend(state, done["q"])}


# ------------------------------------------------------------------------------------------------------ the work
def work(case):
    es = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "rope":
        n = case["tokens"] * case["heads"] * case["dim"]
        times = 2 if case["backward"] else 1
        return {"bytes": times * 2 * n * es + 8 * case["tokens"],
                "flops": times * 3 * case["tokens"] * case["heads"] * case["rot"]}
    length, new = _lengths(case)
    Hq, Hk, D, N = case["heads"], case["kv_heads"], case["dim"], case["page"]
    T = sum(new)
    byte = flop = 0
    if case["kind"] in ("append", "step"):
        byte += T * (2 * Hq + 2 * Hk) * D * es + T * Hk * 2 * D
        flop += 3 * T * (Hq + Hk) * case["rot"] + 4 * T * Hk * D
    if case["kind"] in ("attend", "step"):
        pairs = keys = 0
        for n, q in zip(length, new):
            w = case["window"] or n
            pairs += sum(min(p + 1, w) for p in range(n - q, n))
            keys += n - max(0, n - q + 1 - w)
        byte += T * 2 * Hq * D * es + 4 * T * Hq + keys * Hk * (2 * D + 8.0 / N)
        flop += 4 * pairs * Hq * D
    return {"bytes": byte, "flops": flop}


# ------------------------------------------------------------------------------------------- the 64-bit results
def exact(case, seed):
    """From the definitions, sequence by sequence in 64 bits; a code's value is the number it stands for, unrounded."""
    s = prepare(case, seed)
    turns, f = s["turns"], s["mscale"]

    def spin(x, pos, sign):
        # pairs as complex numbers: times f exp(i angle)
        rot, D = case["rot"], x.shape[-1]
        w = torch.polar(torch.full_like(pos[:, None] * turns, f), sign * 2.0 * math.pi * torch.frac(pos[:, None] * turns))
        order = torch.arange(rot, device="cuda").view(-1, 2) if case["interleaved"] else \
            torch.arange(rot, device="cuda").view(2, -1).t()
        z = torch.view_as_complex(x[..., order].contiguous()) * w[:, None]
        out = x.clone()
        out[..., order.reshape(-1)] = torch.view_as_real(z).reshape(*x.shape[:-1], rot)
        return out

    if case["kind"] == "rope":
        pos = s["positions"].double()
        y = spin(s["x"].detach().double(), pos, 1.0)
        return {"y": y, "dx": spin(s["dy"].double(), pos, -1.0)} if case["backward"] else y

    length, new = _lengths(case)
    N, D, Hq, Hk = case["page"], case["dim"], case["heads"], case["kv_heads"]
    codes_t, top, _, _ = CODES[case["cache"]]
    out = {}
    stored = s["kv"].view(torch.uint8).view(codes_t).float()
    scales = s["scales"].double()
    query = s["q"].double()
    table = s["table"].tolist()
    if case["kind"] in ("append", "step"):
        pos = torch.cat([torch.arange(n - c, n, device="cuda") for n, c in zip(length, new)]).double()
        query = spin(query, pos, 1.0)
        key = spin(s["k"].double(), pos, 1.0)
        x = torch.stack([key, s["v"].double()], 2)                         # (T, kv heads, 2, D)
        value = stored.double() if case["kind"] == "append" and codes_t is not torch.int8 else None
        at = 0
        for r, (n, c) in enumerate(zip(length, new)):
            for w in range((n - c) // N, (n - 1) // N + 1):
                lo, hi = max(n - c, w * N), min(n, w * N + N)
                a, page = at + lo - (n - c), table[r][w]
                part = x[a:a + hi - lo]
                need = torch.exp2(torch.ceil(torch.log2(part.abs().amax((0, 3)) / top)))
                was = scales[page].clone()
                scales[page] = need if lo == w * N else torch.maximum(was, need)
                if value is not None:
                    if lo != w * N:
                        value[page].view(Hk, N, 2, D).mul_((was / scales[page])[:, None, :, None])
                    value[page, :, lo % N:lo % N + hi - lo] = \
                        (part / scales[page][..., None]).transpose(0, 1).reshape(Hk, hi - lo, 2 * D)
            at += c
        out = {"q": query, "kv": value, "scales": scales}
        if case["kind"] == "append":
            return out
        # what attention then reads is what the append rounds to: its own result, from the codes
        return {**out, "o": None, "lse": None}
    o = torch.zeros(sum(new), Hq, D, dtype=torch.float64, device="cuda")
    lse = torch.zeros(sum(new), Hq, dtype=torch.float64, device="cuda")
    at = 0
    for r, (n, c) in enumerate(zip(length, new)):
        pages = torch.tensor(table[r][:-(-n // N)], device="cuda")
        first = n - c - case["window"] + 1 if case["window"] else 0
        keys = torch.arange(max(0, first), n, device="cuda")
        seen = keys[None] <= torch.arange(n - c, n, device="cuda")[:, None]
        if case["window"]:
            seen &= keys[None] > torch.arange(n - c, n, device="cuda")[:, None] - case["window"]
        for h in range(Hk):
            both = stored[pages, h].double().view(-1, N, 2, D) * scales[pages, h][:, None, :, None]
            both = both.view(-1, 2, D)[keys]
            for j in range(h * (Hq // Hk), (h + 1) * (Hq // Hk)):
                z = (query[at:at + c, j] @ both[:, 0].t()) / math.sqrt(D)
                z.masked_fill_(~seen, -math.inf)
                lse[at:at + c, j] = torch.logsumexp(z, 1)
                o[at:at + c, j] = torch.exp(z - lse[at:at + c, j, None]) @ both[:, 1]
        at += c
    return {"o": o, "lse": lse}
