"""Attention of a few query tokens over the paged caches (csrc/tree_attention.hip): trees of drafted tokens over the bf16
and the 8-bit cache, and the 8-bit cache's decode attention, against the definition in 64 bits (oracle/mx_ref.py).

Tolerance of one output element, from the kernel's roundings (u = 2^-24, a = sum_j p_j |v_j| of the element):
  - the result to bf16: 2^-8 |o|;
  - a score: products of bf16 numbers are exact in fp32, their D sums round D times, the scale twice more, and a step in the
    exponent moves p by as much: 2 (D + 3) u (largest sum_d scale |q_d k_d|) a; the factor 2 because numerator and
    denominator both move;
  - exp2 and the rescaling by exp2 of differences of maxima, at most 4 ulp each, one per merge level: 16 u a;
  - p as a bf16 head and a bf16 remainder: 2^-16 a (each rounds to half a step, 2^-8, of what is left);
  - the sums over L tokens, numerator and denominator: 2 L u a.
"""
import ctypes

import pytest
import torch

from nanovllm_hip import _lib
from nanovllm_hip.kernels import (allocate_kvcache_mxfp8, flash_attn_with_kvcache_mxfp8, load_kvcache_mxfp8,
                                  store_kvcache_mxfp8, tree_attention_with_kvcache, tree_mask)
from nanovllm_hip.kernels.attention import flash_attn_varlen_func, flash_attn_with_kvcache
from oracle import mx_ref

gpu = pytest.mark.gpu
BF16, DEV = torch.bfloat16, "cuda"
U = 2.0 ** -24


# ------------------------------------------------------------------ CPU

def test_tree_mask():
    assert tree_mask([]) == [] and tree_mask([-1]) == [1]
    #  0 - 1 - 3
    #    \ 2 - 4,  5 a second root
    assert tree_mask([-1, 0, 0, 1, 2, -1]) == [0b1, 0b11, 0b101, 0b1011, 0b10101, 0b100000]
    chain = tree_mask(list(range(-1, 63)))
    assert chain[62] == 2 ** 63 - 1 and chain[63] == -1   # 64 bits, as int64
    torch.tensor(chain, dtype=torch.int64)
    for bad in ([0], [-1, 1], [-2], [-1] * 65):
        with pytest.raises(AssertionError):
            tree_mask(bad)


def meta_call(cache="bf16", B=2, n=3, Hq=4, Hkv=2, D=64, bs=16, nb=4, **change):
    m = dict(device="meta")
    a = {"q": torch.empty(B, n, Hq, D, dtype=BF16, **m), "lens": torch.empty(B, dtype=torch.int32, **m),
         "table": torch.empty(B, 3, dtype=torch.int32, **m), "mask": torch.empty(B, n, dtype=torch.int64, **m)}
    if cache == "bf16":
        a["k"], a["v"] = (torch.empty(nb, bs, Hkv, D, dtype=BF16, **m) for _ in range(2))
        a["ks"] = a["vs"] = None
    else:
        a["k"], a["v"], a["ks"], a["vs"] = allocate_kvcache_mxfp8(nb, bs, Hkv, D, device="meta")
    a.update({key: f(a) for key, f in change.items()})
    return tree_attention_with_kvcache(a["q"], a["k"], a["v"], a["lens"], a["table"], a["mask"], k_scales=a["ks"],
                                       v_scales=a["vs"])


def test_shapes_through_fake_impl():
    assert meta_call().shape == (2, 3, 4, 64)
    c = allocate_kvcache_mxfp8(4, 16, 2, 128, device="meta")
    o = flash_attn_with_kvcache_mxfp8(torch.empty(2, 1, 4, 128, dtype=BF16, device="meta"), *c,
                                      torch.empty(2, dtype=torch.int32, device="meta"),
                                      torch.empty(2, 3, dtype=torch.int32, device="meta"), causal=True)
    assert o.shape == (2, 1, 4, 128) and o.dtype == BF16
    assert meta_call("mxfp8").dtype == BF16


@pytest.mark.parametrize("cache", ["bf16", "mxfp8"])
@pytest.mark.parametrize("bad", [
    dict(q=lambda a: a["q"].half()), dict(q=lambda a: a["q"][:, :, :3]), dict(q=lambda a: a["q"][..., :32]),
    dict(lens=lambda a: a["lens"].long()), dict(lens=lambda a: a["lens"][:1]), dict(table=lambda a: a["table"].long()),
    dict(table=lambda a: a["table"][:1]), dict(mask=lambda a: a["mask"].int()), dict(mask=lambda a: a["mask"][:, :2]),
    dict(k=lambda a: a["k"][:2]), dict(k=lambda a: a["k"].transpose(1, 2)), dict(v=lambda a: a["v"].view(torch.uint8)),
    dict(ks=lambda a: None if a["ks"] is not None else torch.empty(1, dtype=torch.uint8, device="meta")),
], ids=lambda d: next(iter(d)))
def test_refusals(cache, bad):
    with pytest.raises(AssertionError):
        meta_call(cache, **bad)


def test_at_most_64_query_tokens():
    meta_call(n=64)
    with pytest.raises(AssertionError):
        meta_call(n=65)


def test_abi_refuses_without_launching():
    lib, P, A, E = _lib.lib(), None, ctypes.c_void_p(64), _lib.NVHIP_EINVAL

    def err():
        return lib.nvhip_last_error().decode()

    def call(out=A, q=A, k=A, ks=P, vs=P, bt=A, lens=A, mask=P, B=2, n=3, Hq=4, Hkv=2, D=64, bs=16, nb=4, mb=3, qst=256,
             qsh=64, ost=256, osh=64, scale=0.1, ws=P, size=0):
        return lib.nvhip_tree_attention(out, q, k, A, ks, vs, bt, lens, mask, B, n, Hq, Hkv, D, bs, nb, mb, qst, qsh, ost,
                                        osh, scale, 0, ws, size, P)

    assert call(n=65) == E and "64" in err()
    assert call(n=0) == E and call(Hkv=0) == E and call(bs=0) == E and call(mb=-1) == E and call(B=-1) == E
    assert call(Hq=5) == E and "multiple" in err()
    assert call(D=96) == E and "head_dim" in err()
    assert call(qsh=60) == E and "strides" in err()
    assert call(ost=100) == E and call(qst=260) == E
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert call(scale=scale) == E and "softmax_scale" in err()
    assert call(ks=A) == E and "together" in err()
    assert call(q=ctypes.c_void_p(8)) == E and "aligned" in err()
    assert call(k=P) == E and call(bt=P) == E and call(lens=P) == E and call(out=P) == E and "null" in err()
    assert call(mb=1 << 20, bs=1 << 12) == E and "too large" in err()
    assert call(B=1 << 24, mb=1 << 10, bs=256) == E and "too large" in err()
    size = lib.nvhip_tree_attention_workspace_size(2, 3, 4, 2, 64, 16, 3)
    assert size > 0 and call(ws=ctypes.c_void_p(8), size=size) == E and "aligned" in err()
    assert call(B=0) == _lib.NVHIP_OK and err() == ""
    assert lib.nvhip_tree_attention_workspace_size(0, 3, 4, 2, 64, 16, 3) == 0
    assert lib.nvhip_tree_attention_workspace_size(2, 3, 5, 2, 64, 16, 3) == 0


def test_the_8_bit_cache_has_scales():
    m = dict(device="meta")
    q, lens = torch.empty(2, 1, 4, 64, dtype=BF16, **m), torch.empty(2, dtype=torch.int32, **m)
    table, k = torch.empty(2, 3, dtype=torch.int32, **m), torch.empty(4, 16, 2, 64, dtype=BF16, **m)
    with pytest.raises(AssertionError, match="scales"):
        flash_attn_with_kvcache_mxfp8(q, k, k, None, None, lens, table)


def test_abi_refuses_more_heads_than_offsets_count():
    lib, A = _lib.lib(), ctypes.c_void_p(64)
    Hq = (1 << 16) + 1
    rc = lib.nvhip_tree_attention(A, A, A, A, None, None, A, A, None, 1, 1, Hq, Hq, 64, 64, 1, 1, Hq * 64, 64, Hq * 64, 64,
                                  0.1, 0, None, 0, None)
    assert rc == _lib.NVHIP_EINVAL and "too large" in lib.nvhip_last_error().decode()


# ------------------------------------------------------------------ GPU

class Case:
    """Random inputs of a call. lens: cached tokens of each sequence; mode: "tree" (a random tree), "causal", "all".
    Rows of the caches that no sequence uses, and those behind a sequence's end, are NaN."""

    def __init__(self, lens, n, Hq=16, Hkv=8, D=128, bs=256, cache="mxfp8", mode="tree", seed=0, spare=2):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.n, self.cache, self.mode, self.bs = lens, n, cache, mode, bs
        self.G, self.D = Hq // Hkv, D
        B, need = len(lens), [-(-x // bs) for x in lens]
        nb = sum(need) + spare
        perm, used = torch.randperm(nb, generator=g).tolist(), 0
        self.table = torch.full((B, max(need) + 1), -1, dtype=torch.int32)
        for b, x in enumerate(need):
            self.table[b, :x] = torch.tensor(perm[used:used + x], dtype=torch.int32)
            used += x
        live = torch.zeros(nb, bs, dtype=torch.bool)
        for b, x in enumerate(lens):
            for t in range(x):
                live[self.table[b, t // bs], t % bs] = True
        k, v = (torch.randn(nb, bs, Hkv, D, generator=g) for _ in range(2))
        k[..., ::17] *= 5
        k, v = k.to(BF16), v.to(BF16)
        k[~live], v[~live] = float("nan"), float("nan")
        if cache == "bf16":
            self.caches = [k.to(DEV), v.to(DEV)]
        else:
            self.caches = allocate_kvcache_mxfp8(nb, bs, Hkv, D, device=DEV)
            rows = [x.view(-1, Hkv, D).to(DEV) for x in (k, v)]
            store_kvcache_mxfp8(*rows, *self.caches, torch.arange(nb * bs, dtype=torch.int32, device=DEV))
        self.q = (torch.randn(B, n, Hq, D, generator=g) * 2).to(BF16).to(DEV)
        parents = [[int(torch.randint(-1, max(1, j), (1,), generator=g)) if j else -1 for j in range(n)] for _ in range(B)]
        self.mask = torch.tensor([tree_mask(p) for p in parents], dtype=torch.int64)
        self.scale = None

    def __call__(self):
        lens, table = torch.tensor(self.lens, dtype=torch.int32, device=DEV), self.table.to(DEV)
        if self.mode == "tree":
            more = {} if self.cache == "bf16" else dict(k_scales=self.caches[2], v_scales=self.caches[3])
            return tree_attention_with_kvcache(self.q, *self.caches[:2], lens, table, self.mask.to(DEV), self.scale, **more)
        return flash_attn_with_kvcache_mxfp8(self.q, *self.caches, lens, table, self.scale, causal=self.mode == "causal")

    def visible(self, b):
        L, n = self.lens[b], self.n
        see = torch.ones(n, L, dtype=torch.bool)
        for i in range(n):
            m = int(self.mask[b, i]) if self.mode == "tree" else (2 << i) - 1 if self.mode == "causal" else -1
            for t in range(max(0, L - n), L):
                see[i, t] = bool(m >> (t - (L - n)) & 1)
        return see

    def sequence(self, b):
        if self.cache == "bf16":
            k, v, dim = self.caches[0].cpu().double(), self.caches[1].cpu().double(), 1
        else:
            k, v = (mx_ref.dequantise(self.caches[i].cpu(), self.caches[i + 2].cpu()) for i in (0, 1))
            dim = 2
        rows = [mx_ref.rows_of(x, self.table[b].tolist(), self.lens[b], dim) for x in (k, v)]
        return rows[0][0], rows[1][0], rows[0][1]

    def check(self, out, sequences=None):
        got = out.cpu().double()
        assert got.shape == self.q.shape
        for b in range(len(self.lens)) if sequences is None else sequences:
            L = self.lens[b]
            if L == 0:
                assert bool((got[b] == 0).all())
                continue
            k, v, ok = self.sequence(b)
            o, a, reach = mx_ref.attention(self.q[b].cpu(), k, v, self.visible(b) & ok, self.scale or self.D ** -0.5)
            tol = 2.0 ** -8 * o.abs() + (2 * (self.D + 3) * U * reach[..., None] + 16 * U + 2.0 ** -16 + 2 * L * U) * a
            off = (got[b] - o).abs()
            assert bool((off <= tol).all()), (b, float((off / tol.clamp(min=1e-30)).max()))


CACHES = ["bf16", "mxfp8"]


@gpu
@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("lens,n", [([1], 1), ([7], 7), ([32, 33, 31, 64, 65], 5), ([500], 7), ([300, 0, 1000, 40], 33),
                                     ([257, 64, 2047], 64), ([9] * 70, 3)])
def test_trees(cache, lens, n):
    c = Case(lens, n, cache=cache, seed=n)
    c.check(c(), None if len(lens) < 10 else [0, 31, 63, 64, 69])


@gpu
@pytest.mark.parametrize("mode", ["causal", "all"])
@pytest.mark.parametrize("lens,n", [([1], 1), ([700], 1), ([4, 129, 2, 0, 300], 1), ([1500, 33], 4), ([50, 64, 700], 64)])
def test_decode(mode, lens, n):
    c = Case(lens, n, mode=mode, seed=n + 1)
    c.check(c())


@gpu
@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("Hq,Hkv,D,bs", [(8, 8, 64, 16), (16, 2, 64, 40), (32, 8, 128, 256), (6, 2, 128, 7), (8, 4, 256, 64),
                                          (16, 1, 128, 1), (5, 1, 256, 33), (34, 2, 64, 32), (64, 1, 64, 96)])
def test_heads_dims_and_pages(cache, Hq, Hkv, D, bs):
    c = Case([130, 31, 64], 6, Hq, Hkv, D, bs, cache, seed=Hq + D)
    c.check(c())


@gpu
@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("n,Hq,Hkv,D,bs", [(20, 4, 2, 64, 7), (33, 8, 4, 128, 40), (17, 8, 2, 256, 64), (9, 16, 4, 256, 24),
                                            (64, 6, 2, 64, 64), (64, 2, 2, 128, 16), (11, 6, 1, 128, 192), (50, 3, 1, 256, 1)])
def test_many_rows(cache, n, Hq, Hkv, D, bs):
    """33 rows of a kv head and more, and row counts that leave waves without rows: pages that end inside a step of 64
    tokens, missing pages, contexts shorter than the tree."""
    c = Case([200, 64, 5, 1, 129], n, Hq, Hkv, D, bs, cache, seed=n + D)
    if bs < 64:
        c.table[0, 1] = -1
    c.check(c())


@gpu
@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("lens,n,Hq,Hkv", [
    ([256, 257, 255, 288, 9] * 14, 1, 16, 8),            # 16 rows: contexts of 8 and 9 chunks of 32
    ([512, 513, 511, 544, 30] * 10, 5, 16, 4),           # 32 rows: 16 and 17 chunks
    ([128, 129, 127, 192, 40] * 8, 33, 4, 2),            # 64 rows: 2 and 3 steps of 64
    ([900, 300, 700, 64, 1500, 10, 2000, 400], 33, 16, 8),   # 64 rows: two or three blocks to a unit
])
def test_short_units_and_shared_ones(cache, lens, n, Hq, Hkv):
    """Units on both sides of the length from which they are split, more of them than a block takes."""
    c = Case(lens, n, Hq=Hq, Hkv=Hkv, D=64, bs=64, cache=cache, seed=14)
    c.check(c())


@gpu
@pytest.mark.parametrize("cache", CACHES)
def test_many_rows_over_long_contexts(cache):
    c = Case([4000, 1, 700], 24, Hq=8, Hkv=2, D=64, bs=64, cache=cache, seed=21)
    first = c()
    c.check(first)
    for _ in range(5):
        assert torch.equal(c(), first)


@gpu
@pytest.mark.parametrize("bs", [16, 64])
@pytest.mark.parametrize("what", [float("nan"), float("inf")])
def test_many_rows_do_not_meet_what_they_do_not_see(bs, what):
    for cache in CACHES:
        c = Case([45, 130, 70], 40, Hq=4, Hkv=2, D=64, bs=bs, cache=cache, seed=22)
        clean = c()
        for bad in (3, 38):   # in the tree's first and last step of 64 tokens
            t = 130 - 40 + bad
            page, row = int(c.table[1, t // bs]), t % bs
            if cache == "bf16":
                c.caches[1][page, row] = what
            else:
                c.caches[1].view(torch.uint8)[page, :, row] = 0x7F
        out = c()
        assert torch.equal(out[0], clean[0]) and torch.equal(out[2], clean[2])
        see = c.visible(1)[:, [130 - 40 + 3, 130 - 40 + 38]].any(1)
        assert bool(see.any()) and not bool(see.all())
        for i in range(40):
            if not see[i]:
                assert torch.equal(out[1, i], clean[1, i])
            else:
                assert bool((out[1, i] == what).all()) if cache == "bf16" and what == what else bool(out[1, i].isnan().all())


@gpu
@pytest.mark.parametrize("cache", CACHES)
def test_long_contexts_are_shared_by_blocks(cache):
    c = Case([5000, 1, 3000], 9, Hq=4, Hkv=2, D=64, bs=32, cache=cache, seed=2)
    first = c()
    c.check(first)
    for _ in range(5):  # whichever block merges, the sums are in block order
        assert torch.equal(c(), first)


@gpu
@pytest.mark.parametrize("cache", CACHES)
def test_masks_that_leave_a_row_empty(cache):
    """Sequences that are their tree: a node whose mask names nobody sees nothing; bits from n on are ignored; the bit of
    node 63 is the sign."""
    c = Case([64, 5, 70], 64, Hq=4, Hkv=2, D=64, bs=16, cache=cache, seed=3)
    c.mask[0, 7] = 0
    c.mask[0, 8] = 1 << 20
    c.mask[1, 60] = 0
    c.mask[2, 5] = 0
    out = c()
    c.check(out)
    assert bool((out[0, 7] == 0).all()) and bool((out[1, :59] == 0).all())   # five tokens: nodes 59 .. 63
    assert bool((out[2, 5] != 0).any())
    c = Case([40], 5, Hq=4, Hkv=2, D=64, bs=16, cache=cache, seed=3)
    want = c()
    c.mask |= -1 << 5
    assert torch.equal(c(), want)


@gpu
@pytest.mark.parametrize("mode", ["tree", "causal"])
@pytest.mark.parametrize("bs", [16, 32])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
def test_what_a_row_does_not_see_does_not_reach_it(mode, bs, what):
    """Keys and values of one node that are no numbers: rows that do not see it have their results, rows that do have what
    the definition gives: not a number where the key's are, the infinity (of bf16) where a value is."""
    n, bad = 6, 3
    for cache in (["bf16", "mxfp8"] if mode == "tree" else ["mxfp8"]):
        for which in (0, 1):
            c = Case([45, 70], n, Hq=4, Hkv=2, D=64, bs=bs, cache=cache, mode=mode, seed=5)
            clean = c()
            t = 45 - n + bad
            page, row = int(c.table[0, t // bs]), t % bs
            if cache == "bf16":
                c.caches[which][page, row] = what
            else:
                c.caches[which].view(torch.uint8)[page, :, row] = 0x7F
            out = c()
            assert torch.equal(out[1], clean[1])
            sees = [bool(c.visible(0)[i, t]) for i in range(n)]
            assert any(sees) and not all(sees)
            for i in range(n):
                if not sees[i]:
                    assert torch.equal(out[0, i], clean[0, i])
                elif which == 1 and cache == "bf16" and what == what:
                    assert bool((out[0, i] == what).all())
                elif which == 1 or cache == "mxfp8" or what != what:
                    assert bool(out[0, i].isnan().all())


@gpu
@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("bs", [16, 32, 256])
def test_pages_that_are_missing(cache, bs):
    c = Case([3 * bs + 10, 2 * bs, bs], 3, Hq=4, Hkv=2, D=64, bs=bs, cache=cache, seed=6)
    c.table[0, 1] = -1
    c.table[1, 0] = c.caches[0].shape[0]
    c.table[1, 1] = 2 ** 31 - 1
    c.table[2, 0] = -(2 ** 31)
    out = c()
    c.check(out)
    assert bool((out[1:] == 0).all())


@gpu
@pytest.mark.parametrize("cache", CACHES)
def test_lengths_past_the_block_table(cache):
    """A length of more tokens than the table has pages for is what the table holds; a negative one is 0."""
    c = Case([64, 20], 2, Hq=4, Hkv=2, D=64, bs=32, cache=cache, seed=7)
    c.table = c.table[:, :2].contiguous()
    want = c()
    c.lens = [1000, 20]
    assert torch.equal(c(), want)
    c.lens = [64, -5]
    out = c()
    assert torch.equal(out[0], want[0]) and bool((out[1] == 0).all())


@gpu
@pytest.mark.parametrize("scale", [0.01, 1.0])
def test_scales(scale):
    c = Case([300, 77], 4, cache="mxfp8", seed=8)
    c.scale = scale
    c.check(c())


@gpu
def test_strides_of_q():
    c = Case([100, 45, 33], 4, Hq=4, Hkv=2, D=64, bs=16, seed=9)
    want, q = c(), c.q
    wide = torch.zeros(3, 4, 9, 64, dtype=BF16, device=DEV)      # views of a projection
    wide[:, :, 2:6] = q
    c.q = wide[:, :, 2:6]
    assert torch.equal(c(), want)
    c.q = q.transpose(1, 2).contiguous().transpose(1, 2)          # heads outside tokens
    assert torch.equal(c(), want)
    c.q = torch.zeros(3 * 4 * 4 * 64 + 1, dtype=BF16, device=DEV)[1:].view(3, 4, 4, 64)   # not 16-byte aligned
    c.q.copy_(q)
    assert torch.equal(c(), want)
    odd = torch.zeros(3, 5, 4, 64, dtype=BF16, device=DEV)        # token rows of a longer buffer
    odd[:, :4] = q
    c.q = odd[:, :4]
    assert torch.equal(c(), want)


@gpu
def test_padding_a_batch_changes_nothing():
    c = Case([100, 45, 33, 0, 0], 4, Hq=4, Hkv=2, D=64, bs=16, seed=10)
    out = c()
    assert bool((out[3:] == 0).all())
    c.check(out)
    empty = tree_attention_with_kvcache(c.q[:0], *c.caches[:2], torch.empty(0, dtype=torch.int32, device=DEV),
                                        c.table[:0].to(DEV), c.mask[:0].to(DEV), k_scales=c.caches[2], v_scales=c.caches[3])
    assert empty.shape == (0, 4, 4, 64)


@gpu
@pytest.mark.parametrize("cache", CACHES)
def test_without_workspace(cache):
    """The C ABI with no workspace: one block per unit."""
    c = Case([700, 3, 129], 7, Hq=8, Hkv=2, D=128, bs=64, cache=cache, seed=11)
    B, n, Hq, D = c.q.shape
    out = torch.full_like(c.q, float("nan"))
    lens, table, mask = torch.tensor(c.lens, dtype=torch.int32, device=DEV), c.table.to(DEV), c.mask.to(DEV)
    ptr = [t.data_ptr() for t in c.caches] + ([None, None] if cache == "bf16" else [])
    _lib.check(_lib.lib().nvhip_tree_attention(
        out.data_ptr(), c.q.data_ptr(), *ptr, table.data_ptr(), lens.data_ptr(), mask.data_ptr(), B, n, Hq, 2, D, 64,
        c.caches[0].shape[0], table.shape[1], Hq * D, D, Hq * D, D, D ** -0.5, 0, None, 0, _lib.stream_of(c.q)), "tree")
    c.check(out)


@gpu
def test_workspace_with_anything_in_it():
    """The counts need no initialisation, whatever the workspace held: zeros, ones, a former call's."""
    c = Case([3000, 500], 5, Hq=4, Hkv=2, D=64, bs=32, seed=12)
    B, n, Hq, D = c.q.shape
    lens, table, mask = torch.tensor(c.lens, dtype=torch.int32, device=DEV), c.table.to(DEV), c.mask.to(DEV)
    lib = _lib.lib()
    size = lib.nvhip_tree_attention_workspace_size(B, n, Hq, 2, D, 32, table.shape[1])
    ws = torch.zeros(size, dtype=torch.uint8, device=DEV)
    outs = []
    for fill in (0, 255, 1, None, None, 127):
        if fill is not None:
            ws.fill_(fill)
        out = torch.full_like(c.q, float("nan"))
        _lib.check(lib.nvhip_tree_attention(
            out.data_ptr(), c.q.data_ptr(), *(t.data_ptr() for t in c.caches), table.data_ptr(), lens.data_ptr(),
            mask.data_ptr(), B, n, Hq, 2, D, 32, c.caches[0].shape[0], table.shape[1], Hq * D, D, Hq * D, D, D ** -0.5, 0,
            ws.data_ptr(), size, _lib.stream_of(c.q)), "tree")
        outs.append(out)
    c.check(outs[0])
    assert all(torch.equal(o, outs[0]) for o in outs)


@gpu
def test_two_captured_calls_on_two_streams():
    """Graphs of two calls, replayed at the same time on two streams, and eager calls between: each has its own workspace."""
    a, b = (Case([2500, 900], 6, Hq=8, Hkv=4, D=128, bs=256, cache=cache, seed=13 + i) for i, cache in enumerate(CACHES))
    args = []
    for c in (a, b):
        more = {} if c.cache == "bf16" else dict(k_scales=c.caches[2], v_scales=c.caches[3])
        args.append((c.q, *c.caches[:2], torch.tensor(c.lens, dtype=torch.int32, device=DEV), c.table.to(DEV),
                     c.mask.to(DEV), None, *more.values()))
    want = [tree_attention_with_kvcache(*x) for x in args]
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for x in args:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = tree_attention_with_kvcache(*x)
            out = tree_attention_with_kvcache(*x) if x is args[0] else out   # the second call's workspace is the first's
        graphs.append(graph)
        outs.append(out)
    for _ in range(10):
        for o in outs:
            o.fill_(float("nan"))
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        eager = tree_attention_with_kvcache(*args[1])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(eager, want[1])
    a.check(outs[0])
    b.check(outs[1])


@gpu
def test_new_lengths_in_a_captured_call():
    c = Case([600, 200], 5, Hq=8, Hkv=4, D=128, bs=32, seed=15)
    lens, table, mask = torch.tensor(c.lens, dtype=torch.int32, device=DEV), c.table.to(DEV), c.mask.to(DEV)
    args = (c.q, *c.caches[:2], lens, table, mask, None, *c.caches[2:])
    tree_attention_with_kvcache(*args)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = tree_attention_with_kvcache(*args)
    for new in ([600, 200], [5, 200], [0, 0], [33, 6], [600, 200]):
        lens.copy_(torch.tensor(new))
        graph.replay()
        torch.cuda.synchronize()
        c.lens = new
        c.check(out)


@gpu
def test_offsets_past_32_bits():
    """A page behind 2^32 elements of a cache (2^33 bytes in bf16), of 8 heads x 256 rows x 128."""
    nb, g = 17000, torch.Generator().manual_seed(16)
    pages, L, n = torch.tensor([[16999, 16400]], dtype=torch.int32), 300, 4
    rows = torch.randn(2, 512, 8, 128, generator=g).to(BF16)
    q = torch.randn(1, n, 16, 128, generator=g).to(BF16).to(DEV)
    slots = (pages[0].long()[:, None] * 256 + torch.arange(256)).flatten().to(torch.int32).to(DEV)
    lens, mask = torch.tensor([L], dtype=torch.int32, device=DEV), torch.tensor([tree_mask([-1, 0, 0, 1])], device=DEV)
    see = torch.ones(n, L, dtype=torch.bool)
    see[:, L - n:] = torch.tensor([[bool(m >> j & 1) for j in range(n)] for m in mask[0].tolist()])
    for cache in CACHES:
        if cache == "bf16":
            c = [torch.empty(nb, 256, 8, 128, dtype=BF16, device=DEV) for _ in range(2)]
            for x, r in zip(c, rows):
                x.view(-1, 8, 128)[slots.long()] = r.to(DEV)
            vals, more = [r.double() for r in rows], {}
        else:
            c = [torch.empty(nb, 8, 256, d, dtype=t, device=DEV)
                 for d, t in ((128, torch.float8_e4m3fn), (128, torch.float8_e4m3fn), (4, torch.uint8), (4, torch.uint8))]
            store_kvcache_mxfp8(rows[0].to(DEV), rows[1].to(DEV), *c, slots)
            vals, more = [mx_ref.quantise(r)[0] for r in rows], dict(k_scales=c[2], v_scales=c[3])
        out = tree_attention_with_kvcache(q, c[0], c[1], lens, pages.to(DEV), mask, **more)
        o, a, reach = mx_ref.attention(q[0].cpu(), vals[0][:L], vals[1][:L], see, 128 ** -0.5)
        tol = 2.0 ** -8 * o.abs() + (2 * 131 * U * reach[..., None] + 16 * U + 2.0 ** -16 + 2 * L * U) * a
        assert bool(((out[0].cpu().double() - o).abs() <= tol).all())
        del c


@gpu
def test_a_chain_is_the_decode_attention():
    """A tree without branches over the bf16 cache is flash_attn_with_kvcache's causal call: both near the same numbers."""
    c = Case([300, 33, 1000], 4, Hq=16, Hkv=8, cache="bf16", seed=17)
    c.mask[:] = torch.tensor(tree_mask([-1, 0, 1, 2]))
    c.check(c())
    c.check(flash_attn_with_kvcache(c.q, *c.caches, torch.tensor(c.lens, dtype=torch.int32, device=DEV), c.table.to(DEV),
                                    causal=True))


@gpu
def test_a_prompt_a_chunk_a_decode_step_and_a_tree():
    """The operators as a serving loop runs them: a prompt is stored, a chunk over it reads it back and attends to it, a
    decode step and a tree of drafted tokens follow; every attention against the numbers that the cache holds."""
    g, Hq, Hkv, D, bs = torch.Generator().manual_seed(18), 16, 8, 128, 16
    caches = allocate_kvcache_mxfp8(9, bs, Hkv, D, device=DEV)
    pages = torch.tensor([[4, 0, 7, 2, 8, 1]], dtype=torch.int32)
    table = pages.to(DEV)
    held = [torch.zeros(0, Hkv, D, dtype=torch.float64) for _ in range(2)]
    done = 0
    for step, n in (("chunk", 37), ("chunk", 21), ("decode", 1), ("tree", 7)):
        q, k, v = (torch.randn(n, h, D, generator=g).to(BF16) for h in (Hq, Hkv, Hkv))
        pos = torch.arange(done, done + n)
        slots = (pages[0, pos // bs].long() * bs + pos % bs).to(torch.int32).to(DEV)
        store_kvcache_mxfp8(k.to(DEV), v.to(DEV), *caches, slots)
        done += n
        held = [torch.cat([a, mx_ref.quantise(x)[0]]) for a, x in zip(held, (k, v))]
        lens = torch.tensor([done], dtype=torch.int32, device=DEV)
        masks = tree_mask([-1, 0, 0, 1, 2, -1, 5] if step == "tree" else list(range(-1, n - 1)))
        see = torch.ones(n, done, dtype=torch.bool)
        see[:, done - n:] = torch.tensor([[bool(m >> j & 1) for j in range(n)] for m in masks])
        if step == "chunk":
            cu = torch.tensor([0, done], dtype=torch.int32, device=DEV)
            kk, vv = load_kvcache_mxfp8(*caches, table, cu, done)
            assert torch.equal(kk.cpu().double(), held[0]) and torch.equal(vv.cpu().double(), held[1])
            out = flash_attn_varlen_func(q.to(DEV), kk, vv, n, torch.tensor([0, n], dtype=torch.int32, device=DEV), done,
                                         cu, causal=True)
        elif step == "decode":
            out = flash_attn_with_kvcache_mxfp8(q[None].to(DEV), *caches, lens, table, causal=True)[0]
        else:
            out = tree_attention_with_kvcache(q[None].to(DEV), *caches[:2], lens, table,
                                              torch.tensor([masks], dtype=torch.int64, device=DEV), k_scales=caches[2],
                                              v_scales=caches[3])[0]
        o, a, reach = mx_ref.attention(q, *held, see, D ** -0.5)
        # the prompt's attention rounds p to bf16 once: 2^-8 a
        p_err = 2.0 ** -8 if step == "chunk" else 2.0 ** -16
        tol = 2.0 ** -8 * o.abs() + (2 * (D + 3) * U * reach[..., None] + 16 * U + p_err + 2 * done * U) * a
        assert bool(((out.cpu().double() - o).abs() <= tol).all()), step


@gpu
def test_tensors_on_two_devices_are_refused():
    c = Case([40], 3, Hq=4, Hkv=2, D=64, bs=16)
    lens, table = torch.tensor(c.lens, dtype=torch.int32), c.table.to(DEV)
    with pytest.raises(ValueError, match="tensors on"):
        flash_attn_with_kvcache_mxfp8(c.q, *c.caches, lens, table)
    with pytest.raises(ValueError, match="tensors on"):
        tree_attention_with_kvcache(c.q, *c.caches[:2], lens.to(DEV), table, c.mask, k_scales=c.caches[2],
                                    v_scales=c.caches[3])


@gpu
def test_one_scale_tensor_is_refused():
    c = Case([40], 3, Hq=4, Hkv=2, D=64, bs=16)
    lens, table = torch.tensor(c.lens, dtype=torch.int32, device=DEV), c.table.to(DEV)
    for scales in ((c.caches[2], None), (None, c.caches[3])):
        with pytest.raises(ValueError, match="together"):
            torch.ops.nvhip.tree_attention(c.q, *c.caches[:2], *scales, table, lens, None, 0.1, False)


@gpu
@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("n", [1, 20])
def test_a_cache_without_pages(cache, n):
    """No page is valid: no token takes part, whatever the table and the lengths say, and nothing is read."""
    c = Case([40, 700], n, Hq=8, Hkv=2, D=64, bs=64, cache=cache, seed=13)
    c.caches = [x[:0] for x in c.caches]
    out = c()
    assert out.shape == c.q.shape and bool((out == 0).all())
