"""The operators around an 8-bit KV cache and around drafted tokens, as a serving loop calls them.

Three kinds of case, each one pass:
  kv      the tokens of a step are quantised into the paged cache and the sequences are read back in bf16 (what a prompt
          chunk over a cached prefix needs), 8-bit codes with a power-of-two scale per 32 elements;
  decode  attention of each sequence's last token(s) over that cache;
  tree    attention of a tree of drafted tokens per sequence over the bf16 or the 8-bit cache.
The shapes are those of the package's model configuration (16 query and 8 kv heads of 128, 256-token pages) and, beside
them, the head counts, head dims and page sizes that its tests use.

Format of the 8-bit cache: codes [pages, kv heads, page size, head_dim] e4m3, scales [pages, kv heads, page size,
head_dim / 32] as exponents biased by 127. A block of 32 elements is divided by the least power of two (2^-117 at least)
that brings its largest magnitude to 448 or below, and rounded to the nearest code.
"""
import math
import os
import random
import sys

import torch

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nano-vllm-triton-kernels_amd")
if _PKG not in sys.path:
    sys.path.insert(0, _PKG)

own = False

DEV = "cuda:0"
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
MX = 32            # elements that share a scale
MODEL = {"hq": 16, "hkv": 8, "d": 128, "block": 256}   # the package's model configuration


def listed():
    return [
        # A young sequence gains its next token: the smallest write and the smallest read.
        {"name": "kv_1", "kind": "kv", "seqs": 1, "new": 1, "lo": 33, "hi": 33, "lens": 1, **MODEL},
        # A decode step of 32 requests writes one token each; their (short) sequences are read back.
        {"name": "kv_32", "kind": "kv", "seqs": 32, "new": 1, "lo": 20, "hi": 210, "lens": 2, **MODEL},
        # Chunks of long prompts: each reads back the prefix that it attends to.
        {"name": "kv_chunks", "kind": "kv", "seqs": 5, "new": 250, "lo": 2500, "hi": 9000, "lens": 3, **MODEL},
        # A batch of whole prompts: every token that is read back has just been written.
        {"name": "kv_prompts", "kind": "kv", "seqs": 7, "new": 4096, "lo": 300, "hi": 4096, "lens": 4, **MODEL},
        # One request being decoded: latency.
        {"name": "decode_1", "kind": "decode", "batch": 1, "q_len": 1, "lo": 700, "hi": 700, "lens": 5, **MODEL},
        # The decode step of a server with 32 requests.
        {"name": "decode_32", "kind": "decode", "batch": 32, "q_len": 1, "lo": 512, "hi": 2048, "lens": 6, **MODEL},
        # A large batch with ragged contexts: all cache bandwidth.
        {"name": "decode_250", "kind": "decode", "batch": 250, "q_len": 1, "lo": 40, "hi": 4096, "lens": 7, **MODEL},
        # Two long conversations with few kv heads, small pages and a drafted chain of three tokens.
        {"name": "decode_long", "kind": "decode", "batch": 2, "q_len": 3, "lo": 30000, "hi": 40000, "lens": 8, "hq": 16,
         "hkv": 2, "d": 64, "block": 16},
        # A small tree for one request over the bf16 cache: latency.
        {"name": "tree_1", "kind": "tree", "batch": 1, "nodes": 7, "lo": 500, "hi": 500, "lens": 9, "cache": "bf16", **MODEL},
        # Trees of an odd node count for a few requests over the bf16 cache.
        {"name": "tree_8", "kind": "tree", "batch": 8, "nodes": 33, "lo": 1000, "hi": 4000, "lens": 10, "cache": "bf16", **MODEL},
        # The widest trees for a full batch over the 8-bit cache.
        {"name": "tree_32", "kind": "tree", "batch": 32, "nodes": 64, "lo": 512, "hi": 2048, "lens": 11, "cache": "mxfp8", **MODEL},
        # Four query heads per kv head, heads of 64, small pages, very ragged contexts.
        {"name": "tree_ragged", "kind": "tree", "batch": 13, "nodes": 26, "lo": 30, "hi": 6000, "lens": 12, "cache": "mxfp8",
         "hq": 32, "hkv": 8, "d": 64, "block": 16},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    shape = rng.choice([MODEL, MODEL, {"hq": 32, "hkv": 8, "d": 128, "block": 256}, {"hq": 16, "hkv": 4, "d": 64, "block": 32},
                        {"hq": 16, "hkv": 2, "d": 128, "block": 16}, {"hq": 8, "hkv": 8, "d": 64, "block": 40},
                        {"hq": 8, "hkv": 4, "d": 256, "block": 64}])
    width = shape["hkv"] * shape["d"]
    kind = rng.choice(["kv", "decode", "decode", "tree", "tree"])
    seqs = _log(rng, 1, 200)
    # tokens of all sequences together: the widest listed case of the kind is the most
    most = {"kv": 18_000, "decode": 400_000, "tree": 30_000}[kind] * 1024 // width
    hi = _log(rng, 16, max(16, min(40_000, most // seqs)))
    lo = max(1, int(hi * rng.uniform(0.1, 1.0)))
    case = {"kind": kind, "lo": lo, "hi": hi, "lens": rng.randrange(1, 1 << 30), **shape}
    if kind == "kv":
        return {"seqs": seqs, "new": _log(rng, 1, hi), **case}
    if kind == "decode":
        return {"batch": seqs, "q_len": rng.choice([1, 1, 1, 2, 5]), **case}
    return {"batch": seqs, "nodes": _log(rng, 2, 64 * 2 // max(2, shape["hq"] // shape["hkv"])),
            "cache": rng.choice(["bf16", "mxfp8"]), **case}


def _lens(case):
    """Tokens of each sequence, the step's own among them."""
    rng = random.Random(case["lens"])
    least = case.get("q_len") or case.get("nodes") or 1
    return [max(least, rng.randint(case["lo"], case["hi"])) for _ in range(case.get("seqs") or case["batch"])]


def work(case):
    lens, hkv, d = _lens(case), case["hkv"], case["d"]
    total, mx = sum(lens), d + d // MX
    pages = 4 * sum(-(-n // case["block"]) for n in lens)
    if case["kind"] == "kv":
        new = sum(min(case["new"], n) for n in lens)
        return {"bytes": new * (2 * hkv * (2 * d + mx) + 4) + total * 2 * hkv * (mx + 2 * d) + pages, "flops": 0}
    rows = case.get("q_len") or case["nodes"]
    key = mx if case.get("cache", "mxfp8") == "mxfp8" else 2 * d
    return {"bytes": total * 2 * hkv * key + 2 * len(lens) * rows * case["hq"] * d * 2 + pages,
            "flops": 4 * rows * case["hq"] * d * total}


# ------------------------------------------------------------------ inputs

def _pow2(e):
    """2^e in fp32 for integers -126 <= e <= 127, from the bits."""
    return ((e.to(torch.int32) + 127) << 23).view(F32)


def _quantise(x):
    """[..., d] -> (codes [..., d] e4m3, scales [..., d / 32] uint8)."""
    b = x.float().unflatten(-1, (-1, MX))
    # largest magnitude = mant 2^exp, mant in [0.5, 1); 2^-109 = 0.5 2^-108 gives the least exponent, -117
    mant, exp = torch.frexp(b.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -109))
    e = exp - 9 + (mant > 0.875)
    codes = (b * _pow2(-e)).to(torch.float8_e4m3fn)
    return codes.flatten(-2), (e.squeeze(-1) + 127).to(torch.uint8)


def _dequantise(codes, scales):
    return (codes.float().unflatten(-1, (-1, MX)) * _pow2(scales.to(torch.int32) - 127).unsqueeze(-1)).flatten(-2)


def _values(shape, g, outliers=False):
    """Keys and values as projections give them: near-normal, of keys some channels much larger."""
    x = torch.randn(shape, generator=g, device=DEV, dtype=F32)
    if outliers:
        x = x * torch.where(torch.rand(shape[-2:], generator=g, device=DEV) < 0.04, 6.0, 0.8)
    return x


def _tables(lens, block, g):
    """Scattered pages for each sequence ([seqs, most pages] int32, -1 behind the last one) and how many there are."""
    need = torch.tensor([-(-n // block) for n in lens], device=DEV)
    pages = int(sum(-(-n // block) for n in lens)) + 3
    perm = torch.randperm(pages, generator=g, device=DEV)
    col = torch.arange(int(max(-(-n // block) for n in lens)), device=DEV)
    first = need.cumsum(0) - need
    at = (first[:, None] + col).clamp(max=pages - 1)
    return torch.where(col < need[:, None], perm[at], torch.full_like(at, -1)).to(torch.int32).contiguous(), pages


def prepare(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    lens, hkv, d, block = _lens(case), case["hkv"], case["d"], case["block"]
    table, pages = _tables(lens, block, g)
    s = {"kind": case["kind"], "table": table}
    lens_dev = torch.tensor(lens, dtype=torch.int32, device=DEV)
    if case.get("cache") == "bf16":
        shape = (pages, block, hkv, d)
        s["k"], s["v"] = _values(shape, g, True).to(BF16), _values(shape, g).to(BF16)
    else:
        shape = (pages, hkv, block, d)
        k, v = _values(shape, g).mul_(1.2), _values(shape, g)
        s["k"], s["ks"] = _quantise(k.to(BF16))
        s["v"], s["vs"] = _quantise(v.to(BF16))
    if case["kind"] == "kv":
        new = [min(case["new"], n) for n in lens]
        seq = torch.repeat_interleave(torch.arange(len(lens), device=DEV), torch.tensor(new, device=DEV))
        begin = torch.tensor(new, device=DEV).cumsum(0) - torch.tensor(new, device=DEV)
        pos = torch.arange(sum(new), device=DEV) - begin[seq] + (lens_dev.long() - torch.tensor(new, device=DEV))[seq]
        s["slots"] = (table[seq, pos // block].long() * block + pos % block).to(torch.int32)
        # key and value: views of the projection's output, as the layer hands them over
        qkv = _values((sum(new), 2 * hkv, d), g, True).to(BF16)
        s["key"], s["value"] = qkv[:, :hkv], qkv[:, hkv:]
        s["cu"] = torch.cat([torch.zeros(1, dtype=torch.int32, device=DEV), lens_dev.cumsum(0).to(torch.int32)])
        s["total"] = sum(lens)
        return s
    rows = case.get("q_len") or case["nodes"]
    s["lens"] = lens_dev
    s["q"] = (_values((len(lens), rows, case["hq"], d), g) * 2.0).to(BF16)
    if case["kind"] == "tree":
        # a random tree: node j's parent is one of the nodes before it or, for some, the last accepted token
        parent = (torch.rand(len(lens), rows, generator=g, device=DEV) * (torch.arange(rows, device=DEV) + 1)).long() - 1
        bit = torch.ones((), dtype=torch.int64, device=DEV) << torch.arange(rows, device=DEV)
        mask = bit.expand(len(lens), rows).clone()
        for j in range(1, rows):   # parents come first: one step gives a node all its ancestors
            up = mask.gather(1, parent[:, j:j + 1].clamp(min=0)).squeeze(1)
            mask[:, j] |= torch.where(parent[:, j] >= 0, up, torch.zeros_like(up))
        s["mask"] = mask
    return s


# ------------------------------------------------------------------ one pass

def _scatter(cache, slots, rows):
    """rows [T, heads, n] into cache [pages, heads, page size, n] at the tokens' slots."""
    block = cache.shape[2]
    cache[slots // block, :, slots % block] = rows


def _gather(cache, table, cu, total):
    """The sequences' rows of a cache, one sequence behind the other: [total, heads, n]."""
    t = torch.arange(total, device=table.device)
    seq = torch.searchsorted(cu, t, right=True) - 1
    pos, block = t - cu[seq], cache.shape[2]
    return cache[table[seq, pos // block].long(), :, pos % block]


def _attend(q, k, v, visible):
    """q [B, n, Hq, d], k, v [B, L, Hkv, d] fp32, visible [B, n, L] -> [B, n, Hq, d] bf16; a row that sees nothing is 0."""
    B, n, hq, d = q.shape
    hkv, G = k.shape[2], hq // k.shape[2]
    qh = q.float().view(B, n, hkv, G, d).permute(0, 2, 1, 3, 4).reshape(B, hkv, n * G, d)
    s = torch.matmul(qh, k.permute(0, 2, 3, 1).contiguous()).view(B, hkv, n, G, -1) * d ** -0.5
    s.masked_fill_(~visible[:, None, :, None, :], float("-inf"))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == float("-inf"), torch.zeros_like(m), m))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, hkv, n * G, -1), v.permute(0, 2, 1, 3).contiguous()).view(B, hkv, n, G, d)
    o = o / torch.where(total == 0, torch.ones_like(total), total)
    return o.permute(0, 2, 1, 3, 4).reshape(B, n, hq, d).to(BF16)


def run(s):
    if own:
        from nanovllm_hip import kernels as hip
        if s["kind"] == "kv":
            hip.store_kvcache_mxfp8(s["key"], s["value"], s["k"], s["v"], s["ks"], s["vs"], s["slots"])
            return hip.load_kvcache_mxfp8(s["k"], s["v"], s["ks"], s["vs"], s["table"], s["cu"], s["total"])
        if s["kind"] == "decode":
            return hip.flash_attn_with_kvcache_mxfp8(s["q"], s["k"], s["v"], s["ks"], s["vs"], s["lens"], s["table"],
                                                     causal=True)
        return hip.tree_attention_with_kvcache(s["q"], s["k"], s["v"], s["lens"], s["table"], s["mask"],
                                               k_scales=s.get("ks"), v_scales=s.get("vs"))
    table = s["table"]
    if s["kind"] == "kv":
        slots = s["slots"].long()
        for rows, codes, scales in ((s["key"], s["k"], s["ks"]), (s["value"], s["v"], s["vs"])):
            c, e = _quantise(rows)
            _scatter(codes.view(torch.uint8), slots, c.view(torch.uint8))
            _scatter(scales, slots, e)
        return tuple(_dequantise(_gather(codes.view(torch.uint8), table, s["cu"], s["total"]).view(torch.float8_e4m3fn),
                                 _gather(scales, table, s["cu"], s["total"])).to(BF16)
                     for codes, scales in ((s["k"], s["ks"]), (s["v"], s["vs"])))
    page = table.long().clamp(min=0)
    if "ks" in s:   # [B, pages, Hkv, block, d] -> [B, L, Hkv, d]
        k, v = (_dequantise(c.view(torch.uint8)[page].view(torch.float8_e4m3fn), e[page]).transpose(2, 3).flatten(1, 2)
                for c, e in ((s["k"], s["ks"]), (s["v"], s["vs"])))
    else:
        k, v = s["k"][page].float().flatten(1, 2), s["v"][page].float().flatten(1, 2)
    n, lens, t = s["q"].shape[1], s["lens"].long()[:, None, None], torch.arange(k.shape[1], device=table.device)
    if s["kind"] == "decode":
        visible = t <= lens - n + torch.arange(n, device=table.device)[:, None]
    else:
        node = t - (lens - n)   # the tree is the sequence's last n tokens
        bit = (s["mask"][:, :, None] >> node.clamp(0, n - 1)) & 1
        visible = (t < lens) & ((node < 0) | (bit == 1))
    return _attend(s["q"], k, v, visible)


# ------------------------------------------------------------------ the same in 64 bits

def _code_values():
    """The numbers of the 256 e4m3 codes."""
    out = []
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        v = math.nan if (e, m) == (15, 7) else m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        out.append(-v if c & 128 else v)
    return torch.tensor(out, dtype=F64, device=DEV)


def _stored(codes, scales):
    """What codes and scales stand for."""
    factor = torch.ldexp(torch.ones((), dtype=F64, device=DEV), scales.to(torch.int64) - 127)
    return _code_values()[codes.view(torch.uint8).long()] * factor.repeat_interleave(MX, dim=-1)


def _rounded(x):
    """What x [..., d] stands for once it is stored."""
    b = x.double().unflatten(-1, (-1, MX))
    most = b.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -140)
    scale = torch.exp2(torch.ceil(torch.log2(most / 448) - 1e-12).clamp(min=-117).round())
    y = b / scale
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)) + 1e-12) - 3)
    return (torch.round(y / step) * step * scale).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    lens, block = _lens(case), case["block"]

    def sequence(b, n, x, scales):
        """Tokens 0 .. n - 1 of sequence b of a cache: [n, Hkv, d]."""
        pages = s["table"][b, :-(-n // block)].long()
        if scales is None:
            return x[pages].double().flatten(0, 1)[:n]
        return _stored(x[pages], scales[pages]).transpose(1, 2).flatten(0, 1)[:n]

    if case["kind"] == "kv":
        out, first = ([], []), 0
        for b, n in enumerate(lens):
            new = min(case["new"], n)
            for o, rows, x, scales in ((out[0], s["key"], s["k"], s["ks"]), (out[1], s["value"], s["v"], s["vs"])):
                o.append(sequence(b, n, x, scales)[:n - new])
                o.append(_rounded(rows[first:first + new]))
            first += new
        return tuple(torch.cat(o) for o in out)

    q = s["q"].double()
    rows, G, d = q.shape[1], case["hq"] // case["hkv"], case["d"]
    result = torch.empty_like(q)
    for b, n in enumerate(lens):
        k, v = (sequence(b, n, s[x], s.get(x + "s")) for x in "kv")
        see = torch.ones(rows, n, dtype=torch.bool, device=DEV)
        if case["kind"] == "decode":
            see[:, n - rows:] = torch.ones(rows, rows, dtype=torch.bool, device=DEV).tril()
        else:
            bits = s["mask"][b].tolist()
            see[:, n - rows:] = torch.tensor([[bool(m >> j & 1) for j in range(rows)] for m in bits], device=DEV)
        for h in range(case["hkv"]):
            for j in range(h * G, h * G + G):
                score = (q[b, :, j] @ k[:, h].t().contiguous()) / math.sqrt(d)
                result[b, :, j] = torch.softmax(score.masked_fill(~see, -math.inf), -1) @ v[:, h].contiguous()
    return result
