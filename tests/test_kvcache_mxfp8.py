"""The 8-bit KV cache (csrc/kvcache_mxfp8.hip): what is written, and what is read back, are the numbers of the definition
in 64 bits (oracle/mx_ref.py), exactly: dividing by a power of two is exact, so there is one rounding, and the values are
bf16 numbers. On the CPU: the definition's own error, the refusals of the Python functions (meta tensors) and of the C ABI.
"""
import ctypes

import pytest
import torch

from nanovllm_hip import _lib
from nanovllm_hip.kernels import allocate_kvcache_mxfp8, load_kvcache_mxfp8, store_kvcache_mxfp8
from oracle import mx_ref

gpu = pytest.mark.gpu
BF16 = torch.bfloat16


# ------------------------------------------------------------------ CPU: the definition

def test_error_and_range_of_the_format():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(500, 64, generator=g, dtype=torch.float64) * torch.exp2(torch.randint(-20, 20, (500, 1), generator=g))
    x[0] = 0
    x[1, :32] = 448.0       # the largest code at scale 1
    x[2, :32] = 448.0001    # the next scale
    v, s = mx_ref.quantise(x)
    assert s[1, 0] == 127 and s[2, 0] == 128 and bool((v[0] == 0).all())
    scale = torch.exp2(s.double() - 127).repeat_interleave(32, -1)
    assert bool(((v - x).abs() <= torch.maximum(x.abs() * 2.0 ** -4, scale * 2.0 ** -10)).all())
    assert bool((v.abs() <= 448 * scale).all())
    assert torch.equal(v.to(BF16).double(), v)  # exact in bf16


def test_tiny_blocks_stay_normal_numbers():
    v, s = mx_ref.quantise(torch.full((1, 32), 2.0 ** -126, dtype=torch.float64))
    assert s[0, 0] == 10 and float(v[0, 0]) == 2.0 ** -126
    v, s = mx_ref.quantise(torch.full((1, 32), 2.0 ** -128, dtype=torch.float64))
    assert s[0, 0] == 10 and float(v[0, 0]) == 0.0


# ------------------------------------------------------------------ CPU: refusals

def meta_cache(nb=4, bs=16, Hkv=2, D=64):
    return list(allocate_kvcache_mxfp8(nb, bs, Hkv, D, device="meta"))


def meta_rows(N=5, Hkv=2, D=64, dtype=BF16):
    return torch.empty(N, Hkv, D, dtype=dtype, device="meta")


def test_shapes_through_fake_impl():
    c = meta_cache()
    store_kvcache_mxfp8(meta_rows(), meta_rows(), *c, torch.empty(5, dtype=torch.int32, device="meta"))
    k, v = load_kvcache_mxfp8(*c, torch.empty(3, 2, dtype=torch.int32, device="meta"),
                              torch.empty(4, dtype=torch.int32, device="meta"), 7)
    assert k.shape == v.shape == (7, 2, 64) and k.dtype == v.dtype == BF16


@pytest.mark.parametrize("bad", ["dtype", "mixed", "heads", "dim", "stride", "slots", "slot_type", "code_type",
                                 "scale_type", "scale_shape", "order"])
def test_store_refuses(bad):
    c, k, v = meta_cache(), meta_rows(), meta_rows()
    slots = torch.empty(5, dtype=torch.int32, device="meta")
    if bad == "dtype":
        k, v = meta_rows(dtype=torch.int16), meta_rows(dtype=torch.int16)
    elif bad == "mixed":
        v = meta_rows(dtype=torch.float32)
    elif bad == "heads":
        k, v = meta_rows(Hkv=3), meta_rows(Hkv=3)
    elif bad == "dim":
        c = [torch.empty(4, 2, 16, 96, dtype=torch.float8_e4m3fn, device="meta")] * 2 + \
            [torch.empty(4, 2, 16, 3, dtype=torch.uint8, device="meta")] * 2
        k, v = meta_rows(D=96), meta_rows(D=96)
    elif bad == "stride":
        k = torch.empty(5, 64, 2, dtype=BF16, device="meta").transpose(1, 2)
    elif bad == "slots":
        slots = torch.empty(6, dtype=torch.int32, device="meta")
    elif bad == "slot_type":
        slots = slots.long()
    elif bad == "code_type":
        c[1] = c[1].view(torch.uint8)
    elif bad == "scale_type":
        c[2] = c[2].view(torch.int8)
    elif bad == "scale_shape":
        c[3] = torch.empty(4, 2, 16, 1, dtype=torch.uint8, device="meta")
    elif bad == "order":
        c[0] = torch.empty(4, 16, 2, 64, dtype=torch.float8_e4m3fn, device="meta").transpose(1, 2)
    with pytest.raises(AssertionError):
        store_kvcache_mxfp8(k, v, *c, slots)


@pytest.mark.parametrize("bad", ["table_type", "table_dim", "cu_len", "cu_type", "total"])
def test_load_refuses(bad):
    table, cu, total = (torch.empty(3, 2, dtype=torch.int32, device="meta"), torch.empty(4, dtype=torch.int32, device="meta"),
                        7)
    if bad == "table_type":
        table = table.long()
    elif bad == "table_dim":
        table = table[0]
    elif bad == "cu_len":
        cu = cu[:3]
    elif bad == "cu_type":
        cu = cu.long()
    else:
        total = -1
    with pytest.raises(AssertionError):
        load_kvcache_mxfp8(*meta_cache(), table, cu, total)


def test_no_cpu_fallback():
    c = allocate_kvcache_mxfp8(2, 16, 2, 64)
    rows = torch.zeros(1, 2, 64, dtype=BF16)
    with pytest.raises((NotImplementedError, RuntimeError)):
        store_kvcache_mxfp8(rows, rows, *c, torch.zeros(1, dtype=torch.int32))


def test_abi_refuses_without_launching():
    lib, P, A = _lib.lib(), None, ctypes.c_void_p(64)

    def err():
        return lib.nvhip_last_error().decode()

    def store(caches=(A, A, A, A), k=A, kst=128, nb=4, bs=16, n=5, Hkv=2, D=64, dtype=1):
        return lib.nvhip_store_kvcache_mxfp8(*caches, k, A, kst, 128, A, nb, bs, n, Hkv, D, dtype, P)

    E = _lib.NVHIP_EINVAL
    assert store(D=96) == E and "head_dim" in err()
    assert store(dtype=7) == E and "dtype" in err()
    assert store(kst=100) == E and "stride" in err()
    assert store(bs=0) == E and store(Hkv=0) == E and store(n=-1) == E and store(nb=-1) == E
    assert store(nb=1 << 27, bs=16) == E and "too large" in err()
    assert store(caches=(A, P, A, A)) == E and "null" in err()
    assert store(caches=(A, A, ctypes.c_void_p(72), A)) == E and "aligned" in err()
    assert store(k=P) == E and "null" in err()
    assert store(n=0) == _lib.NVHIP_OK and store(nb=0) == _lib.NVHIP_OK and err() == ""

    def load(out=A, caches=(A, A, A, A), bt=A, cu=A, B=3, total=7, Hkv=2, D=64, bs=16, nb=4, mb=2):
        return lib.nvhip_load_kvcache_mxfp8(out, A, *caches, bt, cu, B, total, Hkv, D, bs, nb, mb, P)

    assert load(D=32) == E and load(total=-1) == E and load(mb=-1) == E and load(B=-1) == E
    assert load(bt=P) == E and "null" in err()
    assert load(cu=P) == E and load(out=P) == E
    assert load(out=ctypes.c_void_p(8)) == E and "aligned" in err()
    assert load(B=0) == E and "no sequence" in err()
    assert load(total=0) == _lib.NVHIP_OK


# ------------------------------------------------------------------ GPU

DEV = "cuda"


def values_of(cache, scales):
    return mx_ref.dequantise(cache.cpu(), scales.cpu())


def same(a, b):
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


def sentinel_cache(nb, bs, Hkv, D):
    """A cache of bytes that no write of these tests leaves by chance everywhere."""
    c = allocate_kvcache_mxfp8(nb, bs, Hkv, D, device=DEV)
    for t in c:
        t.view(torch.uint8).fill_(0x5A)
    return c


def check_store(key, value, c, slots):
    before = [t.clone() for t in c]
    store_kvcache_mxfp8(key, value, *c, slots)
    nb, Hkv, bs, D = c[0].shape
    hit = torch.zeros(nb * bs, dtype=torch.bool)
    sl = slots.cpu().tolist()
    rows = [i for i, s in enumerate(sl) if 0 <= s < nb * bs]
    for s in (sl[i] for i in rows):
        hit[s] = True
    for x, code, scale, b_code, b_scale in ((key, c[0], c[2], before[0], before[2]), (value, c[1], c[3], before[1], before[3])):
        want, byte = mx_ref.quantise(x.cpu()[rows])
        flat = values_of(code, scale).transpose(1, 2).reshape(nb * bs, Hkv, D)
        flat_s = scale.cpu().transpose(1, 2).reshape(nb * bs, Hkv, -1)
        at = torch.tensor([sl[i] for i in rows], dtype=torch.long)
        assert torch.equal(flat_s[at], byte)
        assert same(flat[at], want)
        keep = ~hit  # every other slot as it was
        for new, old in ((code, b_code), (scale, b_scale)):
            n = new.view(torch.uint8).cpu().transpose(1, 2).reshape(nb * bs, -1)
            o = old.view(torch.uint8).cpu().transpose(1, 2).reshape(nb * bs, -1)
            assert torch.equal(n[keep], o[keep])


@gpu
@pytest.mark.parametrize("order", ["by_size", "mixed"])
def test_every_bf16_number(order):
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16)
    if order == "by_size":  # blocks of neighbours: every scale there is
        mag = torch.arange(65536) & 0x7FFF
        bits = bits[torch.argsort(mag, stable=True)]
    else:                   # blocks with numbers of all sizes, infinities and NaN among them
        bits = bits[torch.randperm(65536, generator=torch.Generator().manual_seed(3))]
    x = bits.view(BF16).view(256, 4, 64).to(DEV)
    c = sentinel_cache(20, 16, 4, 64)
    check_store(x, x.flip(0).contiguous(), c, torch.randperm(320, generator=torch.Generator().manual_seed(4))[:256]
                .to(torch.int32).to(DEV))


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_other_types(dtype):
    g = torch.Generator().manual_seed(5)
    lo, hi = (-24, 15) if dtype == torch.float16 else (-149, 127)
    x = torch.randn(200, 2, 128, generator=g, dtype=torch.float64) * \
        torch.exp2(torch.randint(lo, hi, (200, 2, 4, 1), generator=g).double()).expand(-1, -1, -1, 32).reshape(200, 2, 128)
    x = x.to(dtype)
    x[3, 1, 40] = float("inf")
    x[4, 0, 5] = float("nan")
    x[5] = 0
    check_store(x.to(DEV), x.flip(0).to(DEV), sentinel_cache(14, 16, 2, 128),
                torch.randperm(224, generator=g)[:200].to(torch.int32).to(DEV))


@gpu
@pytest.mark.parametrize("N,Hkv,D,bs", [(1, 8, 128, 256), (3, 1, 64, 1), (63, 8, 128, 16), (64, 2, 256, 40),
                                         (100, 3, 64, 7), (513, 8, 128, 256), (700, 2, 256, 33)])
def test_rows_slots_and_padding(N, Hkv, D, bs):
    g = torch.Generator().manual_seed(N)
    nb = (N + bs - 1) // bs + 2
    qkv = torch.randn(N, 4 * Hkv + 1, D, generator=g).to(BF16).to(DEV)   # strided rows: views of a projection
    slots = torch.randperm(nb * bs, generator=g)[:N].to(torch.int32)
    slots[torch.rand(N, generator=g) < 0.1] = -1
    if N > 2:
        slots[1], slots[2] = nb * bs, 2 ** 31 - 1   # outside the cache: skipped
    check_store(qkv[:, Hkv:2 * Hkv], qkv[:, 2 * Hkv:3 * Hkv], sentinel_cache(nb, bs, Hkv, D), slots.to(DEV))


@gpu
@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_rows_that_are_not_aligned(dtype):
    g = torch.Generator().manual_seed(9)
    base = torch.randn(50 * 261 + 5, generator=g).to(dtype).to(DEV)
    key = base[3:].as_strided((50, 2, 64), (261, 64, 1))
    value = base[1:].as_strided((50, 2, 64), (131, 64, 1))
    check_store(key, value, sentinel_cache(4, 16, 2, 64), torch.arange(50, dtype=torch.int32).to(DEV) + 7)


@gpu
def test_nothing_to_store():
    c = sentinel_cache(2, 16, 2, 64)
    before = [t.clone() for t in c]
    empty = torch.empty(0, 2, 64, dtype=BF16, device=DEV)
    store_kvcache_mxfp8(empty, empty, *c, torch.empty(0, dtype=torch.int32, device=DEV))
    none = allocate_kvcache_mxfp8(0, 16, 2, 64, device=DEV)
    one = torch.ones(1, 2, 64, dtype=BF16, device=DEV)
    store_kvcache_mxfp8(one, one, *none, torch.zeros(1, dtype=torch.int32, device=DEV))
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(c, before))
    k, v = load_kvcache_mxfp8(*c, torch.empty(0, 3, dtype=torch.int32, device=DEV),
                              torch.zeros(1, dtype=torch.int32, device=DEV), 0)
    assert k.shape == v.shape == (0, 2, 64)


def filled_cache(nb, bs, Hkv, D, seed):
    """Random codes (NaN ones among them) and scales."""
    g = torch.Generator().manual_seed(seed)
    c = allocate_kvcache_mxfp8(nb, bs, Hkv, D, device=DEV)
    for t in c[:2]:
        t.view(torch.uint8).copy_(torch.randint(0, 256, t.shape, generator=g, dtype=torch.uint8))
    for t in c[2:]:
        t.copy_(torch.randint(10, 248, t.shape, generator=g, dtype=torch.uint8))
    return c


@gpu
@pytest.mark.parametrize("lens,Hkv,D,bs,extra", [([1], 8, 128, 256, 0), ([33, 0, 0, 7], 2, 64, 16, 0),
                                                  ([0, 0, 5, 300, 0], 8, 128, 256, 9), ([700, 64], 1, 256, 40, 3),
                                                  ([3] * 150, 2, 64, 2, 40), ([0], 2, 64, 16, 4)])
def test_read_back(lens, Hkv, D, bs, extra):
    g = torch.Generator().manual_seed(sum(lens))
    need = [-(-n // bs) for n in lens]
    nb = sum(need) + 2
    c = filled_cache(nb, bs, Hkv, D, 1)
    perm, used = torch.randperm(nb, generator=g).tolist(), 0
    table = torch.full((len(lens), max(need) + 1), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(perm[used:used + n], dtype=torch.int32)
        used += n
    if max(lens) > 2 * bs:
        table[lens.index(max(lens)), 1] = -1        # a page that is missing, and one that does not exist
        table[lens.index(max(lens)), 2] = nb
    cu = torch.tensor([0] + lens, dtype=torch.int32).cumsum(0).to(torch.int32)
    total = sum(lens) + extra
    k, v = load_kvcache_mxfp8(*c, table.to(DEV), cu.to(DEV), total)
    for got, code, scale in ((k, c[0], c[2]), (v, c[1], c[3])):
        vals = values_of(code, scale)
        want = torch.zeros(total, Hkv, D, dtype=torch.float64)
        for b, n in enumerate(lens):
            if n:
                rows, ok = mx_ref.rows_of(vals, table[b].tolist(), n, 2)
                want[int(cu[b]):int(cu[b]) + n] = torch.where(ok[:, None, None], rows, torch.zeros_like(rows))
        # random codes and scales reach past bf16's largest number (448 2^120), which no stored block does: infinities
        assert same(got.cpu().double(), want.to(BF16).double())


@gpu
def test_tokens_past_the_block_table_are_zeros():
    c = filled_cache(4, 16, 2, 64, 2)
    k, _ = load_kvcache_mxfp8(*c, torch.tensor([[1]], dtype=torch.int32, device=DEV),
                              torch.tensor([0, 40], dtype=torch.int32, device=DEV), 30)
    assert bool((k[16:] == 0).all()) and same(
        k[:16].cpu().double(), values_of(c[0], c[2])[1].transpose(0, 1).to(BF16).double())


@gpu
def test_offsets_past_32_bits():
    """Codes past 2^32 bytes: 17000 pages of 8 heads x 256 rows x 128."""
    nb = 17000
    c = [torch.empty(nb, 8, 256, d, dtype=t, device=DEV)
         for d, t in ((128, torch.float8_e4m3fn), (128, torch.float8_e4m3fn), (4, torch.uint8), (4, torch.uint8))]
    g = torch.Generator().manual_seed(6)
    x = torch.randn(300, 8, 128, generator=g).to(BF16)
    pages = torch.tensor([[16999, 16400]], dtype=torch.int32)
    t = torch.arange(300)
    slots = (pages[0, t // 256].long() * 256 + t % 256).to(torch.int32)
    store_kvcache_mxfp8(x.to(DEV), x.flip(0).contiguous().to(DEV), *c, slots.to(DEV))
    k, v = load_kvcache_mxfp8(*c, pages.to(DEV), torch.tensor([0, 300], dtype=torch.int32, device=DEV), 300)
    want, _ = mx_ref.quantise(x)
    assert torch.equal(k.cpu().double(), want) and torch.equal(v.cpu().double(), want.flip(0))


@gpu
def test_graph_and_another_stream():
    g = torch.Generator().manual_seed(7)
    c = allocate_kvcache_mxfp8(3, 16, 2, 64, device=DEV)
    x = torch.zeros(5, 2, 64, dtype=BF16, device=DEV)
    slots = torch.tensor([40, 3, -1, 17, 0], dtype=torch.int32, device=DEV)
    table, cu = torch.tensor([[0, 1, 2]], dtype=torch.int32, device=DEV), torch.tensor([0, 48], dtype=torch.int32, device=DEV)

    def step():
        store_kvcache_mxfp8(x, x, *c, slots)
        return load_kvcache_mxfp8(*c, table, cu, 48)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        k, v = step()
    for i in range(4):
        new = torch.randn(5, 2, 64, generator=g).to(BF16)
        x.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        want, _ = mx_ref.quantise(new)
        for row, slot in enumerate([40, 3, -1, 17, 0]):
            if slot >= 0:
                assert torch.equal(k[slot].cpu().double(), want[row]) and torch.equal(v[slot].cpu(), k[slot].cpu())


@gpu
def test_tensors_on_two_devices_are_refused():
    c = allocate_kvcache_mxfp8(2, 16, 2, 64, device=DEV)
    rows = torch.zeros(1, 2, 64, dtype=BF16, device=DEV)
    with pytest.raises(ValueError, match="tensors on"):
        store_kvcache_mxfp8(rows, rows, *c, torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="tensors on"):
        load_kvcache_mxfp8(*c, torch.zeros(1, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32, device=DEV), 1)
