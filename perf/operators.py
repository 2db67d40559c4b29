"""The paged fp8 key/value cache: what is timed of the operators that write it, read it back and attend over it.

Three operators ("op"):
  append   paged_kv_append: keys and values of new tokens into the pages, quantised, a scale per page and head
  read     paged_kv_read: the last tokens of every sequence back as fp16 / bf16
  attend   flash_attention_paged_kv: queries of new tokens against each sequence's pages

A cache is four tensors (k, v, k_descale, v_descale): k and v fp8 [pages, heads_kv, page, head_dim], the descales fp32
[pages, heads_kv], powers of two, x = descale * x8.  Sequence b has seqlens[b] tokens, the n_b new ones (cu_seqlens) its last;
token p lives in slot p % page of page table[b][p // page].
"""
import math
import random

import torch

own = False

FP8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
FP8_MAX = {"e4m3": 448.0, "e5m2": 57344.0}
HALF = {"fp16": torch.float16, "bf16": torch.bfloat16}
E_MIN, E_MAX = -64, 64                                    # exponents a page's scale may have

# the dearest listed case of each kind: operations, bytes, and (plain form) scores held at once
LARGEST_FLOPS = 4.0 * 4 * 32 * 4096 * 4096 / 2 * 128
LARGEST_BYTES = 2.0 ** 28
LARGEST_SCORES = 4.0 * 32 * 4096 * 4096


def _case(name, op, B, Hk, D, page, new, ctx, H=0, half="bf16", fmt="e4m3", causal=True, lse=False, fused=False):
    """new: "n" or "lo-hi" new tokens a sequence; ctx: the same of tokens that it holds before them."""
    return {"name": name, "op": op, "B": B, "H": H, "Hk": Hk, "D": D, "page": page, "new": new, "ctx": ctx, "half": half, "fmt": fmt,
            "causal": causal, "lse": lse, "fused": fused}


def listed():
    return [
        # One token of one sequence goes into the cache: the smallest call, launch latency.
        _case("append_b1_token", "append", 1, 8, 128, 64, "1", "900"),
        # A decode step of a full batch: one token each, at whatever slot of its page.
        _case("append_b128_token", "append", 128, 8, 128, 16, "1", "10-3000"),
        # Prompts of many lengths are written at once, K and V as they lie in the fused projection's output.
        _case("append_b16_prompts", "append", 16, 8, 128, 64, "300-4096", "0", fused=True),
        # A short sequence is read back (to move it, to recompute with it).
        _case("read_b1_333", "read", 1, 8, 128, 16, "333", "0"),
        # A batch of long sequences is read back, narrow heads, the other fp8 format.
        _case("read_b8_s8192_d64", "read", 8, 8, 64, 32, "8192", "0", half="fp16", fmt="e5m2"),
        # One new token against a short chat: latency.
        _case("attend_b1_token_s600", "attend", 1, 8, 128, 16, "1", "600", H=32),
        # The decode step of a batch whose sequences are all of about 8192 tokens.
        _case("attend_b16_token_s8192", "attend", 16, 8, 128, 64, "1", "8000-8191", H=32),
        # The decode step of a large batch of very different lengths, narrow heads, the other fp8 format.
        _case("attend_b64_token_ragged_d64", "attend", 64, 4, 64, 16, "1", "20-8000", H=32, half="fp16", fmt="e5m2"),
        # One token of one very long sequence.
        _case("attend_b1_token_s131072", "attend", 1, 8, 128, 128, "1", "131071", H=32),
        # Four drafted tokens a sequence are checked at once, the widest heads, with the log-sum-exp.
        _case("attend_b8_draft4_s4096_d256", "attend", 8, 4, 256, 32, "4", "3000-4500", H=16, lse=True),
        # A piece of a long prompt against all that came before it.
        _case("attend_b1_chunk1024_s16384", "attend", 1, 8, 128, 64, "1024", "15360", H=32, half="fp16"),
        # Whole prompts, ragged, straight after they were written ("mid_s4096_d128" with shared heads).
        _case("attend_b4_prompts_s4096", "attend", 4, 8, 128, 64, "2500-4096", "0", H=32, fused=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _spread(rng, lo, hi):
    """"n" or "lo-hi" between the two, over the logarithm; a third of the single ones powers of two."""
    a = _log_int(rng, lo, hi)
    if rng.random() < 0.5:
        b = _log_int(rng, lo, hi)
        return "%d-%d" % (min(a, b), max(a, b)) if a != b else str(a)
    return str(min(hi, 2 ** int(round(math.log2(a)))) if rng.random() < 1 / 3 else a)


def draw(rng):
    """One more case of the listed ones' ranges, at most as dear as the dearest of them."""
    while True:
        op = rng.choice(["append", "append", "read", "attend", "attend", "attend", "attend"])
        kind = rng.choice(["token", "token", "draft", "chunk", "prompt"]) if op == "attend" else rng.choice(["token", "prompt", "chunk"])
        Hk, D, page = rng.choice([1, 2, 4, 5, 8]), rng.choice([64, 64, 96, 128, 128, 128, 256]), rng.choice([16, 32, 64, 128])
        group = rng.choice([1, 2, 3, 4, 4, 8])
        if kind == "token":
            B, new, ctx = _log_int(rng, 1, 256), "1", _spread(rng, 1, 32768)
        elif kind == "draft":
            B, new, ctx = _log_int(rng, 1, 64), rng.choice(["2", "3", "4", "1-8"]), _spread(rng, 16, 16384)
        elif kind == "chunk":
            B, new, ctx = _log_int(rng, 1, 16), _spread(rng, 17, 2048), _spread(rng, 1, 16384)
        else:
            B, new, ctx = _log_int(rng, 1, 16), _spread(rng, 2, 4096), "0"
        case = _case("", op, B, Hk, D, page, new, ctx, H=Hk * group if op == "attend" else 0, half=rng.choice(["bf16", "fp16"]),
                     fmt=rng.choice(["e4m3", "e4m3", "e5m2"]), causal=op != "attend" or kind != "draft" or rng.random() < 0.7,
                     lse=op == "attend" and rng.random() < 0.3, fused=op != "read" and rng.random() < 0.3)
        del case["name"]
        if op == "read":
            case["new"], case["ctx"] = _spread(rng, 17, 8192), rng.choice(["0", "0", _spread(rng, 1, 2000)])
        n, lens = _lengths(case)
        w = work(case)
        scores = B * max(n) * max(case["H"], 1) * max(lens)
        gathered = 8.0 * B * max(lens) * Hk * D
        if w["flops"] <= LARGEST_FLOPS and w["bytes"] <= LARGEST_BYTES and gathered <= 2.0 ** 33 and (op != "attend" or scores <= LARGEST_SCORES):
            return case


def _lengths(case):
    """New tokens and lengths (with them) of the sequences: part of the case, the same for every seed."""
    rng = random.Random("%(op)s %(B)d %(new)s %(ctx)s" % case)

    def of(text):
        lo, _, hi = text.partition("-")
        return rng.randint(int(lo), int(hi or lo))

    n = [of(case["new"]) for _ in range(case["B"])]
    return n, [x + of(case["ctx"]) for x in n]


def work(case):
    n, lens = _lengths(case)
    T, Hk, D, H = sum(n), case["Hk"], case["D"], case["H"]
    pages = sum(-(-s // case["page"]) - (s - x) // case["page"] for x, s in zip(n, lens))      # touched by the new tokens
    small = 4 * (2 * case["B"] + pages + 2 * pages * Hk)                     # lengths, page numbers, scales
    if case["op"] != "attend":
        return {"bytes": 2.0 * T * Hk * D * (2 + 1) + small, "flops": 2.0 * T * Hk * D}
    pages = sum(-(-s // case["page"]) for s in lens)
    bytes_ = 2.0 * 2 * T * H * D + 2.0 * sum(lens) * Hk * D + 4 * (2 * case["B"] + pages + 2 * pages * Hk) + (4.0 * T * H if case["lse"] else 0)
    if case["causal"]:
        pairs = sum(x * (s - x) + x * (x + 1) // 2 for x, s in zip(n, lens))
    else:
        pairs = sum(x * s for x, s in zip(n, lens))
    return {"bytes": bytes_, "flops": 4.0 * D * H * pairs}


def _exponent(amax, largest):
    """Smallest e with amax <= largest * 2^e, kept within [E_MIN, E_MAX]."""
    m, x = torch.frexp(amax / largest)                    # amax / largest = m 2^x, 0.5 <= m < 1
    e = torch.where(torch.ldexp(torch.full_like(amax, largest), x - 1) >= amax, x - 1, x)
    return torch.where(amax > 0, e.clamp(E_MIN, E_MAX), E_MIN)


def _pool(case, pages, g):
    """A used pool of pages: fp8 values with outlying channels and tokens of different size, and their scales."""
    Hk, P, D = case["Hk"], case["page"], case["D"]

    def one(outliers):
        x8 = torch.empty(pages, Hk, P, D, dtype=FP8[case["fmt"]], device="cuda")
        d = torch.empty(pages, Hk, device="cuda")
        channel = torch.where(torch.rand(1, Hk, 1, D, generator=g, device="cuda") < outliers, 6.0, 1.0)
        step = max(1, 2 ** 26 // (Hk * P * D))
        for lo in range(0, pages, step):
            n = min(step, pages - lo)
            x = torch.randn(n, Hk, P, D, generator=g, device="cuda") * channel
            x = x * torch.exp(0.3 * torch.randn(n, Hk, P, 1, generator=g, device="cuda"))
            amax = x.abs().amax((2, 3))
            d[lo:lo + n] = torch.ldexp(torch.ones_like(amax), _exponent(amax, FP8_MAX[case["fmt"]]))
            x8[lo:lo + n] = (x / d[lo:lo + n, :, None, None]).to(FP8[case["fmt"]])
        return x8, d

    k, kd = one(0.03)
    v, vd = one(0.0)
    return k, v, kd, vd


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, H, Hk, D, P = case["B"], case["H"], case["Hk"], case["D"], case["page"]
    n, lens = _lengths(case)
    need = [-(-s // P) for s in lens]
    pages = sum(need) + 8                                 # a pool has pages that no sequence of the batch holds
    cache = _pool(case, pages, g)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    width = max(need) + 3
    table = torch.full((B, width), -1, dtype=torch.int32)
    at = 0
    for b, c in enumerate(need):
        table[b, :c] = order[at:at + c]
        at += c
    cu = torch.tensor([0] + n, dtype=torch.int64).cumsum(0).to(torch.int32)
    s = {"case": case, "cache": cache, "table": table.cuda(), "seqlens": torch.tensor(lens, dtype=torch.int32).cuda(), "cu": cu.cuda(),
         "even": len(set(n)) == 1, "tokens": sum(n), "most_new": max(n), "most": max(need) * P, "scale": 1.0 / math.sqrt(D)}
    if case["op"] != "read":
        heads = (H, Hk, Hk) if case["fused"] else ((H,) if case["op"] == "attend" else (Hk, Hk))
        x = torch.randn(s["tokens"], sum(heads), D, generator=g, device="cuda").to(HALF[case["half"]])
        if case["op"] == "append":
            x = x * torch.exp(0.3 * torch.randn(s["tokens"], sum(heads), 1, generator=g, device="cuda")).to(x.dtype)
            parts = x.split(heads, 1)[-2:]                # of the fused projection's output, or of one each
            s["k"], s["v"] = parts if case["fused"] else (t.contiguous() for t in parts)
        else:
            s["q"] = x[:, :H]
    return s


def run(s):
    case = s["case"]
    if own:
        from cutlass_flash_atten_fp8_b200 import flash_attention_paged_kv, paged_kv_append, paged_kv_read
        cu = None if s["even"] else s["cu"]
        if case["op"] == "append":
            paged_kv_append(s["cache"], s["k"], s["v"], s["table"], s["seqlens"], cu_seqlens=cu)
            return list(s["cache"])
        if case["op"] == "read":
            return list(paged_kv_read(s["cache"], s["table"], s["seqlens"], s["tokens"], cu_seqlens=cu, dtype=HALF[case["half"]]))
        return flash_attention_paged_kv(s["q"], s["cache"], s["table"], s["seqlens"], case["causal"], s["scale"], cu_seqlens=cu,
                                        return_lse=case["lse"])
    return {"append": _plain_append, "read": _plain_read, "attend": _plain_attend}[case["op"]](s)


# ---- the plain forms ----------------------------------------------------------------------------------------

def _places(s):
    """Of every new token: its sequence, page and slot, and its position."""
    P, cu, lens = s["case"]["page"], s["cu"].long(), s["seqlens"].long()
    t = torch.arange(s["tokens"], device="cuda")
    b = torch.bucketize(t, cu[1:], right=True)
    pos = t - cu[b] + lens[b] - (cu[b + 1] - cu[b])
    return b, s["table"][b, pos // P].long(), pos % P, pos


def _plain_append(s):
    case, P = s["case"], s["case"]["page"]
    largest, dtype = FP8_MAX[case["fmt"]], FP8[case["fmt"]]
    b, page, slot, pos = _places(s)
    lens, cu = s["seqlens"].long(), s["cu"].long()
    start = lens - (cu[1:] - cu[:-1])                     # the tokens held before
    first = s["table"][torch.arange(case["B"], device="cuda"), start // P].long()
    older = (start % P > 0) & (cu[1:] > cu[:-1])          # the first page touched has older tokens in it
    kept = torch.arange(P, device="cuda")[None] < (start % P)[:, None]
    k8, v8, kd, vd = s["cache"]
    _plain_append_one(k8, kd, s["k"].float(), page, slot, first, older, kept, largest, dtype)
    _plain_append_one(v8, vd, s["v"].float(), page, slot, first, older, kept, largest, dtype)
    return [k8, v8, kd, vd]


def _plain_append_one(x8, descale, x, page, slot, first, older, kept, largest, dtype):
    amax = torch.zeros_like(descale).index_reduce_(0, page, x.abs().amax(2), "amax")
    new = torch.ldexp(torch.ones_like(amax), _exponent(amax, largest))
    rows = first[older]
    old = descale[rows]
    new[rows] = torch.maximum(new[rows], old)
    held = x8[rows]
    again = (held.float() * (old / new[rows])[:, :, None, None]).to(dtype)
    keep = kept[older][:, None, :, None]
    x8[rows] = torch.where(keep, again.float(), held.float()).to(dtype)
    descale[page] = new[page]
    x8[page, :, slot] = (x / new[page][:, :, None]).to(dtype)


def _plain_read(s):
    _, page, slot, _ = _places(s)
    k8, v8, kd, vd = s["cache"]
    dtype = HALF[s["case"]["half"]]
    return [(k8[page, :, slot].float() * kd[page][:, :, None]).to(dtype), (v8[page, :, slot].float() * vd[page][:, :, None]).to(dtype)]


def _plain_attend(s):
    case, (k8, v8, kd, vd) = s["case"], s["cache"]
    B, H, Hk, D, P, G = case["B"], case["H"], case["Hk"], case["D"], case["page"], case["H"] // case["Hk"]
    n, L = s["most_new"], s["most"]
    table = s["table"][:, :L // P].clamp(min=0).long()    # the padding is masked below

    def gathered(x8, d):
        x = x8[table].float() * d[table][..., None, None]                    # [B, pages, Hk, P, D]
        return x.transpose(1, 2).reshape(B, Hk, L, D)

    cu, lens = s["cu"].long(), s["seqlens"].long()
    count = cu[1:] - cu[:-1]
    i = torch.arange(n, device="cuda")
    token = (cu[:-1, None] + i).clamp(max=s["tokens"] - 1)                   # [B, n], those past a sequence's last unused
    q = s["q"].float()[token].reshape(B, n, Hk, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hk, n * G, D)
    score = (q @ gathered(k8, kd).transpose(2, 3)).mul_(s["scale"]).view(B, Hk, n, G, L)
    last = (lens - count)[:, None] + i if case["causal"] else (lens - 1)[:, None].expand(B, n)
    last = torch.minimum(last, (lens - 1)[:, None])
    hidden = torch.arange(L, device="cuda") > last[:, :, None]               # [B, n, L]
    score.masked_fill_(hidden[:, None, :, None], -math.inf)
    m = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(m == -math.inf, 0.0, m)).exp_()
    l = p.sum(-1, keepdim=True)
    o = (p.view(B, Hk, n * G, L) @ gathered(v8, vd)).view(B, Hk, n, G, D)
    o = o / torch.where(l == 0, 1.0, l)
    lse = (m + torch.log(l)).squeeze(-1)
    used = i < count[:, None]
    o = o.permute(0, 2, 1, 3, 4).reshape(B, n, H, D)[used].to(s["q"].dtype)
    lse = lse.permute(0, 2, 1, 3).reshape(B, n, H)[used]
    return [o, lse] if case["lse"] else [o]


# ---- the definitions in 64 bits -------------------------------------------------------------------------------

def exact(case, seed):
    """What run returns, from the definition in 64 bits, a sequence at a time."""
    s = prepare(case, seed)
    n, lens = _lengths(case)
    P, first = case["page"], 0
    table = s["table"].tolist()
    if case["op"] == "append":
        return _exact_append(case, s, n, lens, table)
    parts = ([], [])
    for b in range(case["B"]):
        ids = torch.tensor(table[b][:-(-lens[b] // P)], device="cuda")

        def of(x8, d):                                    # [Hk, lens[b], D]
            x = x8[ids].double() * d[ids].double()[:, :, None, None]
            return x.transpose(0, 1).flatten(1, 2)[:, :lens[b]]

        k, v = of(s["cache"][0], s["cache"][2]), of(s["cache"][1], s["cache"][3])
        if case["op"] == "read":
            for part, x in zip(parts, (k, v)):
                part.append(x[:, lens[b] - n[b]:].transpose(0, 1))
            continue
        q = s["q"][first:first + n[b]].double()
        first += n[b]
        o = torch.empty(q.shape, dtype=torch.float64, device="cuda")
        lse = torch.empty(q.shape[:2], dtype=torch.float64, device="cuda")
        where = torch.arange(lens[b], device="cuda")
        seen = torch.arange(n[b], device="cuda") + (lens[b] - n[b]) if case["causal"] else torch.full((n[b],), lens[b] - 1, device="cuda")
        G = case["H"] // case["Hk"]
        for h in range(case["Hk"]):
            a = torch.einsum("igd,jd->gij", q[:, h * G:(h + 1) * G], k[h]) * s["scale"]
            a = a.masked_fill(where[None, None] > seen[None, :, None], -math.inf)
            lse[:, h * G:(h + 1) * G] = torch.logsumexp(a, -1).t()
            o[:, h * G:(h + 1) * G] = torch.einsum("gij,jd->igd", torch.softmax(a, -1), v[h])
        parts[0].append(o)
        parts[1].append(lse)
    out = [torch.cat(p) for p in parts]
    return out if case["op"] == "read" or case["lse"] else out[:1]


def _exact_append(case, s, n, lens, table):
    P, largest, dtype = case["page"], FP8_MAX[case["fmt"]], FP8[case["fmt"]]
    jobs = []                                             # page, first slot written, first new token, how many
    t = 0
    for b in range(case["B"]):
        p = lens[b] - n[b]
        while p < lens[b]:
            m = min(P - p % P, lens[b] - p)
            jobs.append((table[b][p // P], p % P, t, m))
            p, t = p + m, t + m
    # as many tokens in the pages' order and slots, zeros elsewhere
    job = torch.tensor(jobs, device="cuda")
    slot = torch.arange(P, device="cuda")
    mine = (slot >= job[:, 1:2]) & (slot < job[:, 1:2] + job[:, 3:4])
    token = (job[:, 2:3] + slot - job[:, 1:2]).clamp(0, s["tokens"] - 1)
    past = (slot < job[:, 1:2])[:, None, :, None]
    out = [t.double() for t in s["cache"]]
    for codes, scales, new in ((out[0], out[2], s["k"]), (out[1], out[3], s["v"])):
        step = max(1, 2 ** 25 // (P * case["Hk"] * case["D"]))
        for lo in range(0, len(jobs), step):
            at = slice(lo, lo + step)
            x = new[token[at]].double().transpose(1, 2) * mine[at][:, None, :, None]          # [jobs, Hk, P, D]
            a = x.abs().amax((2, 3))
            # powers of two are exact by ldexp; a logarithm may fall on either side of a whole number
            steps = torch.ldexp(torch.full((), largest, dtype=torch.float64, device="cuda"), torch.arange(E_MIN, E_MAX, device="cuda"))
            d = torch.ldexp(torch.ones_like(a), E_MIN + (a[..., None] > steps).sum(-1))
            before = scales[job[at, 0]]
            old = (job[at, 1] > 0)[:, None]
            d = torch.where(old, torch.maximum(d, before), d)
            held = codes[job[at, 0]]
            # each is a half-precision or fp8 number over a power of two: 32 bits hold it
            again = (held * (before / d)[:, :, None, None]).float().to(dtype).double()
            fresh = (x / d[:, :, None, None]).float().to(dtype).double()
            codes[job[at, 0]] = torch.where(mine[at][:, None, :, None], fresh, torch.where(past[at], again, held))
            scales[job[at, 0]] = d
    return out
