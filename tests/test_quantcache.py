"""Quantised paged KV cache: format and refusals (CPU); write, read-back, page
selection and attention on the GPU against the numpy oracle.

What the format specifies to the bit is compared to the bit.  Attention is held
to a bound made of its roundings: with u = eps/2 of the dtype, O is rounded
once (u |O|), and the attention kernel may round each probability times its
value's step once, which multiplies the code less the codes' middle (u sum_i p_i
step_i |code_i - mid|, plus, in fp16, half the smallest subnormal of a product
scaled to at most 1 for every token); scores and sums are fp32.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import attention as ora
from oracle import quantcache as oq

NAME = {torch.float16: "float16", torch.bfloat16: "bfloat16"}
F16, BF16 = torch.float16, torch.bfloat16


# ------------------------------------------------------------------------ CPU
def test_block_bytes():
    from b200attn import quantcache as qc
    assert qc.block_bytes(128, 16, 4) == 2 * 16 * (64 + 8)
    assert qc.block_bytes(64, 64, 8) == 2 * 64 * (64 + 4)
    for bad in ((96, 16, 4), (128, 24, 4), (128, 16, 5), (0, 0, 0)):
        with pytest.raises(RuntimeError, match="head_dim"):
            qc.block_bytes(*bad)


def test_cache_views_cover_the_block():
    from b200attn import QuantCache
    c = QuantCache.empty(3, 16, 2, 128, bits=4, index=True, device="cpu")
    for i, side in enumerate((0, 1)):
        c.codes(side).fill_(1 + i)
        c.params(side).view(torch.int16).fill_(0x0303 + i * 0x0101)
    n = torch.bincount(c.data.flatten().long(), minlength=5).tolist()
    per = 3 * 2 * 16
    assert n[0] == 0 and n[1:5] == [per * 64, per * 64, per * 8, per * 8]
    assert c.num_pages == 3 and c.num_kv_heads == 2


def test_cache_refuses_wrong_storage():
    from b200attn import QuantCache
    ok = dict(page_size=16, head_dim=64, bits=4, dtype=F16)
    data = torch.zeros(2, 1, 2 * 16 * 36, dtype=torch.uint8)
    QuantCache(data, **ok)
    with pytest.raises(RuntimeError, match="data"):
        QuantCache(data[..., :-1].contiguous(), **ok)
    with pytest.raises(RuntimeError, match="data"):
        QuantCache(data.float(), **ok)
    with pytest.raises(RuntimeError, match="dtype"):
        QuantCache(data, **dict(ok, dtype=torch.float32))
    idx, sc = torch.zeros(2, 1, 2, 64, dtype=torch.int8), torch.zeros(2, 1)
    QuantCache(data, index=idx, index_scale=sc, **ok)
    with pytest.raises(RuntimeError, match="together"):
        QuantCache(data, index=idx, **ok)
    with pytest.raises(RuntimeError, match="index"):
        QuantCache(data, index=idx[:, :, :1], index_scale=sc, **ok)


def test_pool_bookkeeping_and_duplicate_sequences():
    from b200attn.quantcache import QuantPagePool
    pool = QuantPagePool(10, 16, 2, 64, max_seqs=3, max_pages=8, device="cpu", bits=8, index=True)
    pool.reserve(0, 17)
    assert pool.num_free == 8 and pool.cache.index is not None
    k = torch.zeros(2, 2, 1, 64, dtype=F16)
    with pytest.raises(RuntimeError, match="once"):
        pool.append(k, k, seqs=[1, 1])
    with pytest.raises(RuntimeError, match="CUDA"):
        pool.append(k, k, seqs=[1, 2])


def test_entry_points_refuse_on_the_host():
    import b200attn as b
    c = b.QuantCache.empty(4, 16, 2, 64, index=True, device="cpu")
    bt, kl = torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    k = torch.zeros(1, 2, 3, 64, dtype=F16)
    with pytest.raises(RuntimeError, match="CUDA"):
        b.append_paged_quant(k, k, c, bt, kl)
    with pytest.raises(RuntimeError, match="dtype"):
        b.append_paged_quant(k.float(), k.float(), c, bt, kl)
    with pytest.raises(RuntimeError, match="KV heads"):
        b.append_paged_quant(k[:, :1], k[:, :1], c, bt, kl)
    with pytest.raises(RuntimeError, match="both"):
        b.append_paged_quant(k, k[:, :, :2], c, bt, kl)
    with pytest.raises(RuntimeError, match="CUDA"):
        b.read_paged_quant(c, bt, torch.zeros(2, dtype=torch.int32), 0, 0)
    q = torch.zeros(1, 4, 64, dtype=F16)
    with pytest.raises(RuntimeError, match="CUDA"):
        b.decode_paged_quant(q, c, bt, kl)
    with pytest.raises(RuntimeError, match="CUDA"):
        b.select_pages(q, c, bt, kl, 1)


def test_library_refuses_bad_formats_without_a_device():
    from b200attn import _lib
    lib = _lib.load()
    assert lib.b2a_kvq_block_bytes(128, 16, 3) == 0
    assert lib.b2a_kvq_decode_workers(0, 8, 128, 4, 100) == 1
    assert lib.b2a_kvq_decode_workers(1, 8, 128, 4, 16) == 8
    for B, n in ((1, 131072), (64, 32768), (1, 1 << 31)):
        assert 1 <= lib.b2a_kvq_decode_workers(B, 8, 128, 8, n) <= 65535
    assert lib.b2a_kvq_decode_workspace_floats(2, 8, 2, 128, 5) == (5 + 4) * 4 * 129 + 11
    assert lib.b2a_kvq_decode_workspace_floats(2, 8, 2, 128, 3) == (3 + 4) * 4 * 129 + 9


def test_oracle_quantiser_keeps_within_half_a_step():
    """Every finite value reads back within half a step, plus the rounding of the result."""
    rng = np.random.default_rng(0)
    for dtype in ("float16", "bfloat16"):
        for bits in (4, 8):
            x = oq.round_to(rng.standard_normal((50, 128)) * np.exp(rng.standard_normal((50, 1)) * 3), dtype)
            c, s, lo = oq.quantise(x, bits, dtype)
            half = np.repeat(s, 64, -1) * 0.5
            assert (np.abs(oq.values(c, s, lo) - x) <= half * (1 + 1e-5)).all()


# ------------------------------------------------------------------------ GPU
def table_for(lens, page, rng, spare=2, width=None):
    """Random page permutation: (block table int32 [B, max_pages], number of pages)."""
    n = [-(-int(x) // page) for x in lens]
    P = sum(n) + spare
    perm = rng.permutation(P).astype(np.int32)
    bt = np.full((len(lens), max(max(n), 1) if width is None else width), -1, np.int32)
    at = 0
    for b, k in enumerate(n):
        bt[b, :k] = perm[at:at + k]
        at += k
    return bt, P


def np_of(t):
    """float32 values of a 16-bit tensor."""
    return t.float().cpu().numpy()


class Filled:
    """A cache with `lens` tokens per sequence, written through append_paged_quant, and what
    the oracle says it holds."""

    def __init__(self, B, Hkv, D, page, bits, dt, lens, seed=0, index=False, amp=1.0, width=None):
        import b200attn
        rng = np.random.default_rng(seed)
        self.page, self.D, self.bits, self.dt, self.name = page, D, bits, dt, NAME[dt]
        self.lens = list(lens)
        self.bt, P = table_for(lens, page, rng, width=width)
        self.cache = b200attn.QuantCache.empty(P, page, Hkv, D, bits=bits, dtype=dt, index=index)
        # stale bytes in every block, NaN params among them
        self.cache.data.copy_(torch.from_numpy(rng.integers(0, 256, self.cache.data.shape, np.uint8)))
        self.btg = torch.from_numpy(self.bt).cuda()
        self.k, self.v = [], []
        for b, n in enumerate(lens):
            for out, s in ((self.k, 1), (self.v, 2)):
                x = torch.from_numpy(ora.seeded_normal((1, Hkv, max(n, 1), D), seed + 10 * b + s) * amp)
                out.append(x.to(dt)[:, :, :n].cuda())
            if n:
                b200attn.append_paged_quant(self.k[b], self.v[b], self.cache, self.btg[b:b + 1],
                                            torch.zeros(1, dtype=torch.int32, device="cuda"))
        self.kl = torch.tensor(self.lens, dtype=torch.int32, device="cuda")

    def codes(self, b, side):
        """(codes, scale, min) of sequence b: [Hkv, n, ...]."""
        x = np_of((self.k, self.v)[side][b])[0]
        return oq.quantise(x, self.bits, self.name)


def check_attention(f, q, O, L, scale=None, pages=None):
    """O, L against 64 bits within the bound in this file's docstring."""
    u = torch.finfo(f.dt).eps / 2
    Hkv = f.cache.num_kv_heads
    B, H, D = q.shape
    G = H // Hkv
    scale = D ** -0.5 if scale is None else scale
    qn, On, Ln = np_of(q), np_of(O), L.cpu().numpy()
    for b in range(B):
        n = f.lens[b]
        parts = [f.codes(b, s) for s in (0, 1)] if n else None
        for h in range(Hkv):
            heads = slice(h * G, (h + 1) * G)
            if n == 0:
                assert (On[b, heads] == 0).all() and np.isneginf(Ln[b, heads]).all()
                continue
            use = np.arange(n)
            if pages is not None:
                lp = pages[b, h][(pages[b, h] >= 0) & (pages[b, h] * f.page < n)]
                use = np.concatenate([np.arange(p * f.page, min(n, (p + 1) * f.page)) for p in lp]
                                     or [np.zeros(0, int)]).astype(int)
            k = oq.values(*(x[h][use] for x in parts[0]))
            v = oq.values(*(x[h][use] for x in parts[1]))
            Or, Lr = oq.attend(qn[b, heads], k, v, scale)
            if len(use) == 0:
                assert (On[b, heads] == 0).all() and np.isneginf(Ln[b, heads]).all()
                continue
            s = qn[b, heads].astype(np.float64) @ k.T * scale
            e = np.exp(s - s.max(-1, keepdims=True))
            p = e / e.sum(-1, keepdims=True)
            sc = np.repeat(parts[1][1][h][use].astype(np.float64), 64, -1)
            c = parts[1][0][h][use]
            # fp32: scores are sums of D products, off by a few 2^-24 of their size, and the
            # probabilities by as much relatively; 2^-17 of it covers sums and exponentials
            size = (np.abs(qn[b, heads]).astype(np.float64) @ np.abs(k).T * scale).max(-1, keepdims=True)
            fp32 = 2.0 ** -17 * (1 + size)
            sub = 2.0 ** -25 * len(use) * sc.max() * (2 ** f.bits - 1) / e.sum(-1, keepdims=True) * 2
            # p * scale is rounded and multiplies c - mid; mid's own share, p * scale * mid, is
            # kept in fp32, so a rounding weighs |c - mid| and not c (which is less where the
            # codes of a channel are all small, and more where they are large)
            off = np.abs(c.astype(np.float64) - 2 ** (f.bits - 1))
            tol = 1.01 * u * (np.abs(Or) + p @ (sc * off)) + fp32 * (p @ np.abs(v) + p @ (sc * c)) \
                + (sub if f.dt == F16 else 0) + (2.0 ** -25 if f.dt == F16 else 0)
            bad = np.abs(On[b, heads] - Or) > tol
            assert not bad.any(), (b, h, np.abs(On[b, heads] - Or)[bad][:4], tol[bad][:4])
            assert (np.abs(Ln[b, heads] - Lr) <= fp32[:, 0] * 2).all(), (b, h, Ln[b, heads] - Lr)


@pytest.mark.gpu
@pytest.mark.parametrize("D,page,bits,dt,start,T", [
    (128, 16, 4, F16, [0, 5, 31, 16], 1), (128, 16, 4, BF16, [0, 5, 31, 16], 40),
    (64, 32, 8, F16, [1, 0, 63], 77), (64, 64, 4, BF16, [3], 200), (128, 64, 8, BF16, [0, 100], 1),
    (128, 32, 8, F16, [7, 2], 33), (64, 16, 4, F16, [15, 16, 17, 0, 2], 16)], ids=str)
def test_append_is_exact_to_the_bit(D, page, bits, dt, start, T):
    """Codes and params of the written slots are the oracle's; every other byte is as it was."""
    import b200attn
    B, Hkv = len(start), 3
    rng = np.random.default_rng(1)
    bt, P = table_for([s + T for s in start], page, rng)
    cache = b200attn.QuantCache.empty(P, page, Hkv, D, bits=bits, dtype=dt)
    cache.data.copy_(torch.from_numpy(rng.integers(0, 256, cache.data.shape, np.uint8)))
    before = cache.data.cpu().numpy()
    x = [torch.from_numpy(ora.seeded_normal((B, T, Hkv, D), 5 + i)).to(dt).cuda() for i in (0, 1)]
    kl = torch.tensor(start, dtype=torch.int32, device="cuda")
    # a [B, Hkv, T, D] view of token-major rows: strided, not copied
    b200attn.append_paged_quant(x[0].transpose(1, 2), x[1].transpose(1, 2), cache,
                                torch.from_numpy(bt).cuda(), kl)
    assert kl.tolist() == [s + T for s in start]
    want = torch.from_numpy(before.copy())
    shadow = b200attn.QuantCache(want, page_size=page, head_dim=D, bits=bits, dtype=dt)
    for side in (0, 1):
        c, s, lo = oq.quantise(np_of(x[side]), bits, NAME[dt])      # [B, T, Hkv, ...]
        if bits == 4:
            c = c[..., ::2] | c[..., 1::2] << 4
        par = torch.from_numpy(np.stack((s, lo), -1)).to(dt)
        for b in range(B):
            for t in range(T):
                pos = start[b] + t
                pg, sl = int(bt[b, pos // page]), pos % page
                shadow.codes(side)[pg, :, sl] = torch.from_numpy(c[b, t])
                shadow.params(side)[pg, :, sl] = par[b, t]
    assert torch.equal(cache.data.cpu(), want)
    assert b200attn.device_error_flags() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, BF16], ids=str)
@pytest.mark.parametrize("bits", [4, 8])
def test_append_of_extreme_values(dt, bits):
    """Constants, zeros, the type's extremes, subnormals, NaN and infinities."""
    import b200attn
    big, tiny = torch.finfo(dt).max, torch.finfo(dt).smallest_normal
    sub = tiny * torch.finfo(dt).eps
    g = torch.Generator().manual_seed(0)
    rows = [torch.zeros(128), torch.full((128,), 3.25), torch.full((128,), -big),
            torch.linspace(-big, big, 128), torch.linspace(0, big, 128),
            torch.randn(128, generator=g) * tiny, torch.randint(0, 9, (128,), generator=g) * sub,
            torch.cat((torch.full((64,), big), torch.full((64,), float("nan")))),
            torch.randn(128, generator=g), torch.randn(128, generator=g), torch.randn(128, generator=g),
            torch.linspace(-1, 1, 128) * big]
    rows[9][70], rows[10][3] = float("inf"), -float("inf")
    x = torch.stack(rows).to(dt)
    T = len(rows)
    cache = b200attn.QuantCache.empty(1, 16, 1, 128, bits=bits, dtype=dt, index=True)
    bt = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    kl = torch.zeros(1, dtype=torch.int32, device="cuda")
    xg = x[None, None].cuda()
    b200attn.append_paged_quant(xg, xg, cache, bt, kl)
    c, s, lo = oq.quantise(np_of(x), bits, NAME[dt])
    got = oq.unpack(cache.data.cpu().numpy(), 16, 128, bits, NAME[dt])
    for side in (0, 1):
        for a, w in zip(got[side], (c, s, lo)):
            np.testing.assert_array_equal(a[0, 0, :T], w)
    K, V = b200attn.read_paged_quant(cache, bt, torch.tensor([0, T], dtype=torch.int32, device="cuda"), T, T)
    np.testing.assert_array_equal(np_of(K)[:, 0], oq.read_back(c, s, lo, NAME[dt]))
    np.testing.assert_array_equal(np_of(V)[:, 0], oq.read_back(c, s, lo, NAME[dt]))
    # a finite group stays finite (a linspace over all of bf16's range passes fp32's itself)
    fine = np.isfinite(np_of(x).reshape(T, 2, 64)).all(-1)
    assert fine[:3].all() and fine[-1].all() and (np.isfinite(np_of(K).reshape(T, 2, 64)).all(-1) == fine).all()
    assert np.isnan(cache.index_scale.item()) and not cache.index.any()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, BF16], ids=str)
@pytest.mark.parametrize("bits", [4, 8])
def test_append_of_wide_ranges(dt, bits):
    """Groups whose range passes the type's largest value (and in bf16 fp32's), from one side
    and the other, beside groups of ordinary size in the same rows: which steps are rounded
    down and which up, and the codes that go with them."""
    import b200attn
    big, T = torch.finfo(dt).max, 96
    g = torch.Generator().manual_seed(3)
    x = torch.rand(T, 128, generator=g, dtype=torch.float64) * 2 - 1
    side = torch.linspace(0, 1, T, dtype=torch.float64)[:, None]
    x = torch.where(x > 0, x * (1 - side), x * side) * big     # one bound at the largest or less
    x[::3, 5], x[1::3, 9] = big, -big
    x[::4, 64:] = torch.randn(T // 4, 64, generator=g, dtype=torch.float64)
    x = x.to(dt)
    cache = b200attn.QuantCache.empty(6, 16, 1, 128, bits=bits, dtype=dt, index=True)
    bt = torch.arange(6, dtype=torch.int32, device="cuda")[None]
    kl = torch.zeros(1, dtype=torch.int32, device="cuda")
    xg = x[None, None].cuda()
    b200attn.append_paged_quant(xg, xg.flip(2), cache, bt, kl)
    got = oq.unpack(cache.data.cpu().numpy(), 16, 128, bits, NAME[dt])
    for s, y in ((0, x), (1, x.flip(0))):
        for a, w in zip(got[s], oq.quantise(np_of(y), bits, NAME[dt])):
            np.testing.assert_array_equal(a.reshape(T, -1), w)


@pytest.mark.gpu
@pytest.mark.parametrize("D,page,bits,dt", [(128, 16, 4, F16), (64, 32, 8, BF16), (64, 64, 4, F16),
                                            (128, 64, 8, F16), (128, 32, 4, BF16)], ids=str)
def test_read_back(D, page, bits, dt):
    """Whole sequences and ranges of them, packed; other rows of `out` are left as they were."""
    import b200attn
    lens = [1, 100, 0, 64, 37]
    f = Filled(5, 2, D, page, bits, dt, lens, seed=3)
    want = [[oq.read_back(*f.codes(b, s), NAME[dt]).transpose(1, 0, 2) if n else np.zeros((0, 2, D))
             for b, n in enumerate(lens)] for s in (0, 1)]
    cu = np.concatenate(([0], np.cumsum(lens))).astype(np.int32)
    out = b200attn.read_paged_quant(f.cache, f.btg, torch.from_numpy(cu).cuda(), int(cu[-1]), max(lens))
    for s in (0, 1):
        np.testing.assert_array_equal(np_of(out[s]), np.concatenate(want[s]))
    # ranges, into rows that leave gaps: 7 free rows at the end
    start = [0, 33, 0, 15, 36]
    take = [1, 40, 0, 49, 1]
    cu = np.concatenate(([0], np.cumsum(take))).astype(np.int32)
    total = int(cu[-1]) + 7
    out = [torch.full((total, 2, D), 9.0, dtype=dt, device="cuda") for _ in (0, 1)]
    res = b200attn.read_paged_quant(f.cache, f.btg, torch.from_numpy(cu).cuda(), total, 49,
                                    start=torch.tensor(start, dtype=torch.int32, device="cuda"), out=out)
    assert res[0] is out[0]
    for s in (0, 1):
        w = np.concatenate([want[s][b][start[b]:start[b] + take[b]] for b in range(5)])
        np.testing.assert_array_equal(np_of(out[s])[:-7], w)
        assert (out[s][-7:] == 9).all()
    assert b200attn.device_error_flags() == 0


@pytest.mark.gpu
def test_bad_pages_and_lengths_are_flagged():
    import b200attn
    dt = F16
    cache = b200attn.QuantCache.empty(4, 16, 1, 64, dtype=dt, index=True)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    k = torch.ones(3, 1, 20, 64, dtype=dt, device="cuda")
    b200attn.device_error_flags()
    # sequence 0: negative length; 1: second page missing; 2: page number past the pool
    bt = i32([0, 1], [2, -1], [7, 3])
    b200attn.append_paged_quant(k, k, cache, bt, i32(-4, 0, 0), advance=False)
    assert b200attn.device_error_flags() & 4
    got = cache.params(0)[:, 0, :, 0, 1].cpu()
    assert (got[2] == 1).all() and (got[3, :4] == 1).all() and not got[3, 4:].any() and not got[:2].any()
    # reading: a missing page reads as zero
    out = b200attn.read_paged_quant(cache, i32([2, -1]), i32(0, 20), 20, 20)
    assert b200attn.device_error_flags() & 2
    assert (out[0][:16] == 1).all() and not out[0][16:].any()
    # a longer sequence than max_len, and a prefix sum past total: not read
    keep = [torch.full((20, 1, 64), 5.0, dtype=dt, device="cuda") for _ in (0, 1)]
    b200attn.read_paged_quant(cache, i32([2, 3]), i32(0, 20), 20, 19, out=keep)
    assert b200attn.device_error_flags() & 8 and (keep[0] == 5).all()
    b200attn.read_paged_quant(cache, i32([2, 3]), i32(0, 21), 20, 21, out=keep)
    assert b200attn.device_error_flags() & 8 and (keep[0] == 5).all()
    # attention and selection: page 0 instead, and a length that the table cannot hold
    q = torch.ones(1, 1, 64, dtype=dt, device="cuda")
    b200attn.decode_paged_quant(q, cache, i32([9]), i32(5))
    assert b200attn.device_error_flags() & 2
    b200attn.decode_paged_quant(q, cache, i32([2]), i32(17))
    assert b200attn.device_error_flags() & 2
    assert b200attn.select_pages(q, cache, i32([2]), i32(17), 1).tolist() == [[[0]]]
    assert b200attn.device_error_flags() & 2
    O, L = b200attn.decode_paged_quant(q, cache, i32([2]), i32(-1))
    assert not O.any() and torch.isneginf(L).all()
    assert b200attn.device_error_flags() & 2


DECODE = [
    # B, H, Hkv, D, page, bits, dtype, lens
    (4, 32, 8, 128, 16, 4, F16, [1, 15, 16, 17]),
    (3, 8, 2, 128, 16, 4, BF16, [1000, 64, 513]),
    (4, 3, 3, 64, 32, 8, F16, [0, 63, 300, 64]),
    (2, 14, 2, 64, 64, 4, BF16, [129, 4000]),
    (2, 5, 1, 128, 64, 8, F16, [777, 65]),
    (1, 16, 2, 128, 32, 8, BF16, [2050]),
    (3, 8, 1, 64, 16, 4, F16, [5000, 0, 31]),
    (2, 6, 2, 128, 32, 4, F16, [333, 1]),
    (1, 8, 8, 64, 16, 8, BF16, [48]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,H,Hkv,D,page,bits,dt,lens", DECODE, ids=str)
def test_decode(B, H, Hkv, D, page, bits, dt, lens):
    import b200attn
    f = Filled(B, Hkv, D, page, bits, dt, lens, seed=7)
    q = torch.from_numpy(ora.seeded_normal((B, H, D), 9)).to(dt).cuda()
    for splits in (None, 1, 3, 40):
        O, L = b200attn.decode_paged_quant(q, f.cache, f.btg, f.kl, splits=splits)
        check_attention(f, q, O, L)
    O4, L4 = b200attn.decode_paged_quant(q[:, :, None], f.cache, f.btg, f.kl, scale=0.3)
    assert O4.shape == (B, H, 1, D) and L4.shape == (B, H, 1)
    check_attention(f, q, O4[:, :, 0], L4[:, :, 0], scale=0.3)
    again = b200attn.decode_paged_quant(q, f.cache, f.btg, f.kl)
    first = b200attn.decode_paged_quant(q, f.cache, f.btg, f.kl)
    assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])
    assert b200attn.device_error_flags() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, BF16], ids=str)
@pytest.mark.parametrize("amp", [1e-4, 30.0])
def test_decode_amplitudes(dt, amp):
    """Small and large keys and values: what the probabilities are scaled by follows the data."""
    import b200attn
    f = Filled(2, 2, 128, 16, 4, dt, [900, 70], seed=17, amp=amp)
    q = torch.from_numpy(ora.seeded_normal((2, 8, 128), 19)).to(dt).cuda()
    O, L = b200attn.decode_paged_quant(q, f.cache, f.btg, f.kl, scale=0.01)
    check_attention(f, q, O, L, scale=0.01)


@pytest.mark.gpu
@pytest.mark.parametrize("D,page,bits,G", [(128, 64, 4, 8), (64, 16, 8, 4), (128, 32, 8, 7)])
def test_decode_of_a_few_tokens(D, page, bits, G):
    """Sequences so short that a channel's codes may all be small: there the outputs' rounding
    errors are those of codes less the middle."""
    import b200attn
    lens = [2, 3, 5, 1, 0, 4, 2, 64] * 4
    f = Filled(len(lens), 3, D, page, bits, F16, lens, seed=97)
    q = torch.from_numpy(ora.seeded_normal((len(lens), 3 * G, D), 99)).half().cuda()
    O, L = b200attn.decode_paged_quant(q, f.cache, f.btg, f.kl)
    check_attention(f, q, O, L)


@pytest.mark.gpu
def test_decode_of_growing_values():
    """Values whose step grows by 2^8 along the sequence, and shrinks again."""
    import b200attn
    f = Filled(1, 1, 64, 16, 8, F16, [640], seed=27)
    ramp = torch.exp2(8 - (torch.arange(640) - 320).abs() / 40)[None, None, :, None].cuda()
    f.v[0] = (f.v[0].float() * ramp).half()
    b200attn.append_paged_quant(f.k[0], f.v[0], f.cache, f.btg,
                                torch.zeros(1, dtype=torch.int32, device="cuda"))
    q = torch.from_numpy(ora.seeded_normal((1, 4, 64), 29)).half().cuda()
    for splits in (1, 2):
        O, L = b200attn.decode_paged_quant(q, f.cache, f.btg, f.kl, splits=splits)
        check_attention(f, q, O, L)


@pytest.mark.gpu
def test_decode_propagates_nan_and_hides_none():
    """A token with a NaN in K makes its heads' outputs NaN (not zero); other heads keep theirs."""
    import b200attn
    f = Filled(2, 2, 64, 16, 4, F16, [300, 20], seed=37)
    q = torch.from_numpy(ora.seeded_normal((2, 4, 64), 39)).half().cuda()
    want = b200attn.decode_paged_quant(q, f.cache, f.btg, f.kl)
    k = f.k[0].clone()
    k[0, 1, 250, 3] = float("nan")
    b200attn.append_paged_quant(k, f.v[0], f.cache, f.btg[:1],
                                torch.zeros(1, dtype=torch.int32, device="cuda"))
    for splits in (1, 5):
        O, L = b200attn.decode_paged_quant(q, f.cache, f.btg, f.kl, splits=splits)
        assert O[0, 2:].isnan().all() and L[0, 2:].isnan().all()
        assert torch.isfinite(O[0, :2]).all() and torch.isfinite(O[1]).all()
        torch.testing.assert_close(O[1], want[0][1], atol=2e-3, rtol=2e-3)


@pytest.mark.gpu
@pytest.mark.parametrize("B,H,Hkv,D,page,bits,dt,lens,top", [
    (3, 8, 2, 128, 16, 4, F16, [1000, 64, 513], 5), (2, 6, 2, 64, 32, 8, BF16, [1, 3000], 24),
    (2, 8, 1, 64, 16, 4, BF16, [0, 9000], 100), (1, 5, 5, 128, 64, 8, F16, [4100], 1),
    (1, 4, 1, 128, 16, 4, F16, [5000], 400), (4, 7, 1, 64, 16, 8, F16, [16, 17, 2000, 1999], 125)], ids=str)
def test_index_select_and_sparse_decode(B, H, Hkv, D, page, bits, dt, lens, top):
    import b200attn
    f = Filled(B, Hkv, D, page, bits, dt, lens, seed=47, index=True)
    G = H // Hkv
    idx, isc = f.cache.index.cpu().numpy(), f.cache.index_scale.cpu().numpy()
    q = torch.from_numpy(ora.seeded_normal((B, H, D), 49)).to(dt).cuda()
    pages = b200attn.select_pages(q, f.cache, f.btg, f.kl, top)
    got = pages.cpu().numpy()
    for b, n in enumerate(lens):
        count = -(-n // page)
        phys = f.bt[b, :count]
        if n:
            c, s, lo = f.codes(b, 0)
            k = oq.read_back(c, s, lo, NAME[dt])
        for h in range(Hkv):
            for p in range(count):
                ci, si = oq.bounds(k[h, p * page:min(n, (p + 1) * page)])
                np.testing.assert_array_equal(idx[phys[p], h], ci)
                assert isc[phys[p], h] == si
            want = oq.select(np_of(q)[b, h * G:(h + 1) * G], idx[phys, h], isc[phys, h], count, top)
            np.testing.assert_array_equal(got[b, h], want)
    for splits in (None, 1, 7):
        O, L = b200attn.decode_paged_quant(q, f.cache, f.btg, f.kl, pages=pages, splits=splits)
        check_attention(f, q, O, L, pages=got)
    assert b200attn.device_error_flags() == 0


@pytest.mark.gpu
def test_index_follows_single_appends():
    """Token by token, through a page that held an older sequence's keys."""
    import b200attn
    B, Hkv, D, page = 2, 2, 128, 16
    f = Filled(B, Hkv, D, page, 4, BF16, [3 * page, page], seed=57, index=True)
    kl = torch.tensor([0, 14], dtype=torch.int32, device="cuda")      # sequence 0 starts again
    lens = [0, 14]
    held = [np.zeros((Hkv, 0, D), np.float32), oq.read_back(*f.codes(1, 0), "bfloat16")[:, :14]]
    bt = torch.cat((f.btg[:, :1], f.btg[:1, 1:2].expand(2, 1)), 1)
    bt[1, 1] = f.cache.num_pages - 1
    bt = bt.contiguous()
    for step in range(18):                # up to the table's 32 tokens
        x = torch.from_numpy(ora.seeded_normal((B, Hkv, 1, D), 100 + step)).to(BF16)
        b200attn.append_paged_quant(x.cuda(), x.cuda(), f.cache, bt, kl)
        y = oq.read_back(*oq.quantise(np_of(x), 4, "bfloat16"), "bfloat16")
        for b in range(B):
            held[b] = np.concatenate((held[b], y[b]), 1)
            lens[b] += 1
            p = (lens[b] - 1) // page
            for h in range(Hkv):
                ci, si = oq.bounds(held[b][h, p * page:])
                np.testing.assert_array_equal(f.cache.index[bt[b, p], h].cpu().numpy(), ci)
                assert f.cache.index_scale[bt[b, p], h].item() == si
    assert kl.tolist() == lens


@pytest.mark.gpu
def test_select_ties_and_non_finite_scores():
    """Equal pages: the lowest are taken.  A page or query that is not finite is never left out."""
    import b200attn
    D, page, n = 64, 16, 40
    cache = b200attn.QuantCache.empty(n, page, 1, D, dtype=F16, index=True)
    cache.index.fill_(5)
    cache.index_scale.fill_(0.25)
    bt = torch.arange(n, dtype=torch.int32, device="cuda")[None].contiguous()
    kl = torch.tensor([n * page - 3], dtype=torch.int32, device="cuda")
    q = torch.from_numpy(ora.seeded_normal((1, 4, D), 3)).half().cuda()
    pick = lambda k: b200attn.select_pages(q, cache, bt, kl, k)[0, 0].tolist()  # noqa: E731
    assert pick(4) == [0, 1, 2, n - 1]
    cache.index_scale[20], cache.index_scale[7] = float("nan"), 100.0
    assert pick(3) == ([7, 20, n - 1] if (q.float().sum(-1) > 0).any() else [0, 20, n - 1])
    assert pick(n + 5) == list(range(n)) + [-1] * 5
    q[0, 1, 3] = float("nan")                                      # every page scores +infinity
    assert pick(4) == [0, 1, 2, 3]
    q.zero_()
    assert pick(2) == [20, n - 1]


@pytest.mark.gpu
def test_page_lists_of_the_caller():
    """Negative and out-of-range entries are skipped wherever they stand; none left: O = 0."""
    import b200attn
    f = Filled(1, 2, 64, 16, 8, F16, [200], seed=67)
    q = torch.from_numpy(ora.seeded_normal((1, 4, 64), 69)).half().cuda()
    lists = np.array([[[-1, 3, -7, 12, 0, 99, -1, -1, 5], [-1] * 9]], np.int32)
    for splits in (1, 2, 9):
        O, L = b200attn.decode_paged_quant(q, f.cache, f.btg, f.kl, pages=torch.from_numpy(lists).cuda(),
                                           splits=splits)
        check_attention(f, q, O, L, pages=lists)
    assert b200attn.device_error_flags() == 0


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Pages whose bytes lie past 4 GiB of the pool."""
    import b200attn
    Hkv, D, page = 8, 128, 64
    per = Hkv * 2 * page * (64 + 8)
    P = (1 << 32) // per + 40
    cache = b200attn.QuantCache(torch.empty(P, Hkv, per // Hkv, dtype=torch.uint8, device="cuda"),
                                page_size=page, head_dim=D, bits=4, dtype=F16)
    n = 300
    bt = torch.arange(P - 1, P - 6, -1, dtype=torch.int32, device="cuda")[None].contiguous()
    kl = torch.zeros(1, dtype=torch.int32, device="cuda")
    k, v = (torch.from_numpy(ora.seeded_normal((1, Hkv, n, D), s)).half().cuda() for s in (1, 2))
    b200attn.append_paged_quant(k, v, cache, bt, kl)
    c = [oq.quantise(np_of(x)[0], 4, "float16") for x in (k, v)]
    out = b200attn.read_paged_quant(cache, bt, torch.tensor([0, n], dtype=torch.int32, device="cuda"), n, n)
    for s in (0, 1):
        np.testing.assert_array_equal(np_of(out[s]).transpose(1, 0, 2), oq.read_back(*c[s], "float16"))
    q = torch.from_numpy(ora.seeded_normal((1, 32, D), 3)).half().cuda()
    f = Filled.__new__(Filled)
    f.cache, f.lens, f.page, f.bits, f.dt, f.name, f.k, f.v = cache, [n], page, 4, F16, "float16", [k], [v]
    O, L = b200attn.decode_paged_quant(q, cache, bt, kl)
    check_attention(f, q, O, L)


@pytest.mark.gpu
def test_strided_and_misaligned_inputs():
    """Views of one fused projection, and rows that are not 16-byte aligned (copied)."""
    import b200attn
    f = Filled(2, 2, 64, 16, 4, F16, [50, 33], seed=77)
    qkv = torch.from_numpy(ora.seeded_normal((2, 8 + 4, 64), 5)).half().cuda()
    q = qkv[:, :8]
    want = b200attn.decode_paged_quant(q.contiguous(), f.cache, f.btg, f.kl)
    got = b200attn.decode_paged_quant(q, f.cache, f.btg, f.kl)
    assert torch.equal(want[0], got[0])
    odd = torch.zeros(2 * 8 * 64 + 1, dtype=F16, device="cuda")[1:].view(2, 8, 64)
    odd.copy_(q)
    assert torch.equal(want[0], b200attn.decode_paged_quant(odd, f.cache, f.btg, f.kl)[0])
    one = torch.empty_strided((1, 8, 64), (13, 64, 1), dtype=F16, device="cuda")  # a stride nobody uses
    one.copy_(q[:1])
    assert torch.equal(want[0][:1], b200attn.decode_paged_quant(one, f.cache, f.btg[:1], f.kl[:1])[0])
    wide = torch.zeros(2, 8, 64, 2, dtype=F16, device="cuda")[..., 0]             # rows not contiguous
    wide.copy_(q)
    assert torch.equal(want[0], b200attn.decode_paged_quant(wide, f.cache, f.btg, f.kl)[0])
    k = qkv[:, 8:10, None]
    a, b = f.cache.data.clone(), f.cache.data.clone()
    kl = f.kl.clone()
    for data, x in ((a, k), (b, k.contiguous())):
        c = b200attn.QuantCache(data, page_size=16, head_dim=64, bits=4, dtype=F16)
        b200attn.append_paged_quant(x, x, c, f.btg, kl - 1, advance=False)
    assert torch.equal(a, b) and not torch.equal(a, f.cache.data)


@pytest.mark.gpu
def test_refusals_on_the_device():
    import b200attn as b
    c = b.QuantCache.empty(4, 16, 1, 64, dtype=F16)
    i32 = dict(dtype=torch.int32, device="cuda")
    bt, kl = torch.zeros(1, 4, **i32), torch.ones(1, **i32)
    q = torch.zeros(1, 9, 64, dtype=F16, device="cuda")
    with pytest.raises(RuntimeError, match="at most 8"):
        b.decode_paged_quant(q, c, bt, kl)
    q = q[:, :2]
    with pytest.raises(RuntimeError, match="dtype"):
        b.decode_paged_quant(q.bfloat16(), c, bt, kl)
    with pytest.raises(RuntimeError, match="index"):
        b.select_pages(q, c, bt, kl, 2)
    with pytest.raises(RuntimeError, match="scale"):
        b.decode_paged_quant(q, c, bt, kl, scale=-1.0)
    with pytest.raises(RuntimeError, match="splits"):
        b.decode_paged_quant(q, c, bt, kl, splits=0)
    with pytest.raises(RuntimeError, match="pages"):
        b.decode_paged_quant(q, c, bt, kl, pages=torch.zeros(1, 2, 3, **i32))
    with pytest.raises(RuntimeError, match="block_table"):
        b.decode_paged_quant(q, c, bt.long(), kl)
    with pytest.raises(RuntimeError, match="kv_lens"):
        b.decode_paged_quant(q, c, bt, torch.ones(2, **i32))
    with pytest.raises(RuntimeError, match="max_pages"):
        b.decode_paged_quant(q, c, bt[:, :0], kl)
    e = b.decode_paged_quant(q[:0], c, bt[:0], kl[:0])
    assert e[0].shape == (0, 2, 64)
    K, V = b.read_paged_quant(c, bt, torch.zeros(2, **i32), 0, 0)
    assert K.shape == (0, 1, 64)
    b.append_paged_quant(torch.zeros(1, 1, 0, 64, dtype=F16, device="cuda"),
                         torch.zeros(1, 1, 0, 64, dtype=F16, device="cuda"), c, bt, kl)
    assert kl.tolist() == [1]


@pytest.mark.gpu
def test_serving_run_together():
    """Prompt, chunked prefill over the read-back cache, decode steps, sparse decode: a
    QuantPagePool as a server uses it, next to attention over the read-back values."""
    import b200attn
    from b200attn.quantcache import QuantPagePool
    B, H, Hkv, D, page, dt = 3, 8, 2, 128, 16, BF16
    pool = QuantPagePool(80, page, Hkv, D, max_seqs=B, max_pages=24, dtype=dt, bits=8, index=True)
    k, v = (torch.from_numpy(ora.seeded_normal((B, Hkv, 70, D), s)).to(dt).cuda() for s in (1, 2))
    pool.append(k, v)
    k1, v1 = (torch.from_numpy(ora.seeded_normal((2, Hkv, 21, D), s)).to(dt).cuda() for s in (3, 4))
    pool.append(k1, v1, seqs=[2, 0])
    assert pool.lengths() == [91, 70, 91] and pool.kv_lens.tolist() == [91, 70, 91]
    K, V, cu, most = pool.read()
    assert cu.tolist() == [0, 91, 161, 252] and most == 91
    # the last 21 tokens' queries of sequences 0 and 2, as a prefill chunk over the cache
    K2, V2, cu2, _ = pool.read(seqs=[0, 2])
    assert torch.equal(K2, torch.cat((K[:91], K[161:]))) and torch.equal(V2[91:], V[161:])
    Q = torch.from_numpy(ora.seeded_normal((42, H, D), 5)).to(dt).cuda()
    cq = torch.tensor([0, 21, 42], dtype=torch.int32, device="cuda")
    O, L = b200attn.forward_varlen(Q, K2, V2, cq, cu2, 21, causal=True)
    # the last query of each chunk sees all keys: the decode step of the same query agrees
    Od, Ld = pool.decode(Q[[20, 41]].contiguous(), seqs=[0, 2])
    torch.testing.assert_close(Od.float(), O[[20, 41]].float(), atol=1e-2, rtol=2e-2)
    torch.testing.assert_close(Ld, L[:, [20, 41]].t(), atol=1e-2, rtol=1e-3)
    all_pages = pool.decode(Q[[20, 41]].contiguous(), seqs=[0, 2], top_k=6)
    torch.testing.assert_close(all_pages[0].float(), Od.float(), atol=1e-2, rtol=2e-2)
    few = pool.decode(Q[:3].contiguous(), top_k=2)
    assert torch.isfinite(few[0].float()).all()
    pool.release(1)
    assert pool.lengths()[1] == 0 and pool.kv_lens.tolist()[1] == 0
    O1, L1 = pool.decode(Q[:3].contiguous())
    assert not O1[1].any() and torch.isneginf(L1[1]).all()
    assert b200attn.device_error_flags() == 0


@pytest.mark.gpu
def test_captured_step_and_side_streams():
    """A captured step (append, select, decode) replays on new inputs, next to a second graph of
    the same cache layout and eager calls on another stream."""
    import b200attn
    B, H, Hkv, D, page = 2, 8, 2, 64, 16
    fs = [Filled(B, Hkv, D, page, 4, F16, [600, 90], seed=87 + i, index=True, width=48) for i in (0, 1)]
    graphs = []
    for f in fs:
        # pages for growth past the last full one
        f.x = torch.zeros(B, Hkv, 1, D, dtype=F16, device="cuda")
        f.q = torch.zeros(B, H, D, dtype=F16, device="cuda")

        def step(f=f):
            b200attn.append_paged_quant(f.x, f.x, f.cache, f.btg, f.at, advance=False)
            pages = b200attn.select_pages(f.q, f.cache, f.btg, f.kl, 9)
            return b200attn.decode_paged_quant(f.q, f.cache, f.btg, f.kl, pages=pages, splits=3) + [pages]

        f.at = f.kl - 1                      # overwrite each sequence's last token
        f.step = step
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            f.out = step()
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in fs]
    for it in range(3):
        for f, g, s in zip(fs, graphs, streams):
            f.x.copy_(torch.from_numpy(ora.seeded_normal((B, Hkv, 1, D), 200 + it)).half())
            f.q.copy_(torch.from_numpy(ora.seeded_normal((B, H, D), 300 + it)).half())
            s.wait_stream(torch.cuda.current_stream())
        for f, g, s in zip(fs, graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for f in fs:
            got = [t.clone() for t in f.out]
            want = f.step()
            torch.cuda.synchronize()
            for a, w in zip(got, want):
                assert torch.equal(a, w)
            for b in range(B):
                f.k[b][0, :, -1] = f.x[b, :, 0]
                f.v[b][0, :, -1] = f.x[b, :, 0]
            check_attention(f, f.q, got[0], got[1], pages=got[2].cpu().numpy())
    assert b200attn.device_error_flags() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("count,top", [(2048, 100), (2049, 100), (9000, 333), (16385, 16), (20000, 3000)], ids=str)
def test_select_of_long_tables(count, top):
    """Tables past the sizes at which the selection changes its form; many pages share bounds,
    so that ties cross every boundary inside it."""
    import b200attn
    D, page, P = 64, 16, 97
    rng = np.random.default_rng(count)
    cache = b200attn.QuantCache.empty(P, page, 1, D, dtype=F16, index=True)
    bounds = np.sort(rng.integers(-127, 128, cache.index.shape).astype(np.int8), axis=2)  # min <= max
    cache.index.copy_(torch.from_numpy(bounds))
    cache.index_scale.copy_(torch.from_numpy(rng.uniform(0.01, 1, (P, 1)).astype(np.float32)))
    table = rng.integers(0, P, (1, count)).astype(np.int32)
    kl = torch.tensor([count * page - 5], dtype=torch.int32, device="cuda")
    q = torch.from_numpy(ora.seeded_normal((1, 3, D), 3)).half().cuda()
    got = b200attn.select_pages(q, cache, torch.from_numpy(table).cuda(), kl, top)[0, 0].cpu().numpy()
    idx, sc = cache.index.cpu().numpy()[table[0], 0], cache.index_scale.cpu().numpy()[table[0], 0]
    np.testing.assert_array_equal(got, oq.select(np_of(q)[0], idx, sc, count, top))


@pytest.mark.gpu
@pytest.mark.parametrize("workers", [1, 2, 5, 64])
def test_runs_over_many_sequences(workers, monkeypatch):
    """Few warps, so that a run crosses long, short and empty sequences and all their heads,
    and its page look-ups cross their ends."""
    import b200attn
    from b200attn import quantcache as qc
    lens = [0, 700, 3, 0, 0, 64, 65, 1, 1500, 16, 17, 0, 130] + [5, 0, 33] * 9 + [400, 0]
    f = Filled(len(lens), 2, 64, 16, 4, F16, lens, seed=107)
    q = torch.from_numpy(ora.seeded_normal((len(lens), 6, 64), 109)).half().cuda()
    lib = __import__("b200attn._lib", fromlist=["load"]).load()
    monkeypatch.setattr(qc, "_plan", lambda B, H, Hkv, D, bits, most, splits: (
        workers, lib.b2a_kvq_decode_workspace_floats(B, H, Hkv, D, workers)))
    O, L = b200attn.decode_paged_quant(q, f.cache, f.btg, f.kl)
    check_attention(f, q, O, L)
    # the same through page lists, some of whose sequences are empty
    lists = np.full((len(lens), 2, 9), -1, np.int32)
    for b, n in enumerate(lens):
        for h in range(2):
            got = np.random.default_rng(b).permutation(max(-(-n // 16), 1))[:9]
            lists[b, h, :len(got)] = got
    O, L = b200attn.decode_paged_quant(q, f.cache, f.btg, f.kl, pages=torch.from_numpy(lists).cuda())
    check_attention(f, q, O, L, pages=lists)
    assert b200attn.device_error_flags() == 0


@pytest.mark.gpu
def test_chained_steps_without_waiting():
    """Forty serving steps back to back (append with advance, select, decode), whose kernels may
    start before the one ahead has ended, give what the same steps give one by one."""
    import b200attn
    B, H, Hkv, D, page, n = 3, 8, 2, 128, 16, 40
    xs = [torch.from_numpy(ora.seeded_normal((B, Hkv, 1, D), 400 + i)).bfloat16().cuda() for i in range(n)]
    qs = [torch.from_numpy(ora.seeded_normal((B, H, D), 500 + i)).bfloat16().cuda() for i in range(n)]

    def run(wait):
        f = Filled(B, Hkv, D, page, 8, BF16, [500, 31, 7], seed=97, index=True, width=40)
        # pages for what is appended: behind the pool's used ones
        f.cache = b200attn.QuantCache.empty(200, page, Hkv, D, bits=8, dtype=BF16, index=True)
        bt = torch.arange(3 * 40, dtype=torch.int32, device="cuda").view(3, 40)
        kl = torch.zeros(B, dtype=torch.int32, device="cuda")
        for b in range(B):
            b200attn.append_paged_quant(f.k[b], f.v[b], f.cache, bt[b:b + 1], kl[b:b + 1])
        outs = []
        for x, q in zip(xs, qs):
            b200attn.append_paged_quant(x, x, f.cache, bt, kl)
            if wait:
                torch.cuda.synchronize()
            pages = b200attn.select_pages(q, f.cache, bt, kl, 6)
            if wait:
                torch.cuda.synchronize()
            outs.append(b200attn.decode_paged_quant(q, f.cache, bt, kl, pages=pages) + [pages])
            if wait:
                torch.cuda.synchronize()
        assert kl.tolist() == [500 + n, 31 + n, 7 + n]
        return outs

    for a, b in zip(run(False), run(True)):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


@pytest.mark.gpu
def test_ctypes_and_cpython_bindings_agree(monkeypatch):
    import b200attn
    from b200attn import quantcache as qc
    f = Filled(2, 2, 64, 16, 4, F16, [90, 40], seed=117, index=True)
    q = torch.from_numpy(ora.seeded_normal((2, 4, 64), 119)).half().cuda()
    x = torch.from_numpy(ora.seeded_normal((2, 2, 3, 64), 120)).half().cuda()
    cu = torch.tensor([0, 90, 130], dtype=torch.int32, device="cuda")

    def all_of():
        b200attn.append_paged_quant(x, x, f.cache, f.btg, f.kl - 3, advance=False)
        pages = b200attn.select_pages(q, f.cache, f.btg, f.kl, 2)
        return (b200attn.read_paged_quant(f.cache, f.btg, cu, 130, 90) + [pages]
                + b200attn.decode_paged_quant(q, f.cache, f.btg, f.kl, pages=pages, scale=0.5))

    first = all_of()
    for name in ("_append", "_read", "_select", "_decode"):
        monkeypatch.setattr(qc, name, getattr(qc, name + "_ct"))
    for a, b in zip(first, all_of()):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_value_nan_stays_in_its_channels():
    """A NaN in one group of one token's V: those 64 channels of its KV head's outputs only."""
    import b200attn
    f = Filled(1, 2, 128, 16, 8, BF16, [130], seed=127)
    v = f.v[0].clone()
    v[0, 1, 77, 100] = float("nan")
    b200attn.append_paged_quant(f.k[0], v, f.cache, f.btg, torch.zeros(1, dtype=torch.int32, device="cuda"))
    q = torch.from_numpy(ora.seeded_normal((1, 4, 128), 129)).bfloat16().cuda()
    for splits in (1, 3):
        O, L = b200attn.decode_paged_quant(q, f.cache, f.btg, f.kl, splits=splits)
        assert O[0, 2:, 64:].isnan().all() and torch.isfinite(O[0, 2:, :64]).all()
        assert torch.isfinite(O[0, :2]).all() and torch.isfinite(L).all()


@pytest.mark.gpu
def test_queries_of_any_size():
    """Query amplitudes over the type's range: they are scaled by powers of two inside."""
    import b200attn
    for dt, amps in ((F16, (1e-6, 1e-3, 1e3)), (BF16, (1e-30, 1e-9, 1e9, 1e25))):
        f = Filled(1, 1, 64, 16, 8, dt, [200], seed=137)
        for amp in amps:
            q = (torch.from_numpy(ora.seeded_normal((1, 3, 64), 139)) * amp).to(dt).cuda()
            q[0, 1] = 0
            scale = 0.125 / amp
            O, L = b200attn.decode_paged_quant(q, f.cache, f.btg, f.kl, scale=scale)
            check_attention(f, q, O, L, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, BF16], ids=str)
def test_many_sequences(dt):
    """More (sequence, KV head)s than warps run at a time, empty sequences among them; and
    more sequences than a warp looks at in one go."""
    import b200attn
    B, Hkv, D, page = 700, 4, 64, 16
    rng = np.random.default_rng(3)
    lens = rng.integers(0, 140, B)
    lens[::7] = 0
    bt, P = table_for(lens, page, rng)
    cache = b200attn.QuantCache.empty(P, page, Hkv, D, bits=8, dtype=dt)
    k, v = (torch.from_numpy(ora.seeded_normal((B, Hkv, 140, D), s)).to(dt).cuda() for s in (1, 2))
    btg = torch.from_numpy(bt).cuda()
    kl = torch.from_numpy(lens.astype(np.int32)).cuda()
    q = torch.from_numpy(ora.seeded_normal((B, 8, D), 3)).to(dt).cuda()
    for b in range(B):  # each sequence its own length
        if lens[b]:
            b200attn.append_paged_quant(k[b:b + 1, :, :lens[b]], v[b:b + 1, :, :lens[b]], cache, btg[b:b + 1],
                                        torch.zeros(1, dtype=torch.int32, device="cuda"))
    f = Filled.__new__(Filled)
    f.cache, f.lens, f.page, f.bits, f.dt, f.name = cache, lens.tolist(), page, 8, dt, NAME[dt]
    f.k = [k[b:b + 1, :, :lens[b]] for b in range(B)]
    f.v = [v[b:b + 1, :, :lens[b]] for b in range(B)]
    for splits in (None, 1):
        O, L = b200attn.decode_paged_quant(q, cache, btg, kl, splits=splits)
        check_attention(f, q, O, L)
    assert b200attn.device_error_flags() == 0


def check_own_steps(f, q, O, L):
    """check_attention's bound with nothing in it that another token's or channel group's step
    enters except by its weight.  A product p * step is rounded to fp16 in a unit that brings the
    largest product of its head and group to 2^7 or more, so where it falls into the subnormals
    half of their spacing is 2^-25 * 2^-7 of that largest product (and it multiplies |code - mid|,
    at most 2^(bits - 1)).  No unit is below 2^-125, of weights that are at most 2^-16: with 2^-25
    that is 2^-134, half of bf16's smallest number."""
    u = torch.finfo(f.dt).eps / 2
    Hkv = f.cache.num_kv_heads
    G = q.shape[1] // Hkv
    qn, On, Ln = np_of(q), np_of(O), L.cpu().numpy()
    mid = 2 ** (f.bits - 1)
    for b, n in enumerate(f.lens):
        K, V = (f.codes(b, s) for s in (0, 1))
        for h in range(Hkv):
            heads = slice(h * G, (h + 1) * G)
            k, v = oq.values(*(x[h] for x in K)), oq.values(*(x[h] for x in V))
            Or, Lr = oq.attend(qn[b, heads], k, v, f.D ** -0.5)
            s = qn[b, heads].astype(np.float64) @ k.T * f.D ** -0.5
            p = np.exp(s - Lr[:, None])
            sc, c = np.repeat(V[1][h].astype(np.float64), 64, -1), V[0][h].astype(np.float64)
            most = (p[:, :, None] * sc).max(1)       # of each head and channel's group
            fp32 = 2.0 ** -17 * (1 + (np.abs(qn[b, heads]).astype(np.float64) @ np.abs(k).T
                                      * f.D ** -0.5).max(-1, keepdims=True))
            tol = 1.01 * u * (np.abs(Or) + p @ (sc * np.abs(c - mid))) \
                + fp32 * (p @ np.abs(v) + p @ (sc * c)) + 2.0 ** -32 * n * mid * most \
                + (2.0 ** -25 if f.dt == F16 else 2.0 ** -133)
            bad = ~(np.abs(On[b, heads] - Or) <= tol)
            assert not bad.any(), (b, h, np.abs(On[b, heads] - Or)[bad][:4], tol[bad][:4])
            assert (np.abs(Ln[b, heads] - Lr) <= fp32[:, 0] * 2).all()


def with_values(f, v=None, k=None):
    """Sequence 0 of f written again, with other values or keys."""
    import b200attn
    f.v[0], f.k[0] = f.v[0] if v is None else v, f.k[0] if k is None else k
    b200attn.append_paged_quant(f.k[0], f.v[0], f.cache, f.btg,
                                torch.zeros(1, dtype=torch.int32, device="cuda"))


RANGE = [(128, 4, F16, 4), (128, 8, BF16, 4), (128, 4, BF16, 8), (128, 8, F16, 6), (64, 4, BF16, 1),
         (64, 8, F16, 8)]


@pytest.mark.gpu
@pytest.mark.parametrize("D,bits,dt,G", RANGE, ids=str)
@pytest.mark.parametrize("at", [0, 300, 511])
def test_a_large_value_without_weight(D, bits, dt, G, at):
    """One token whose values are very much larger than all others' and whose score leaves it
    next to no weight: the others' share of the output is as exact as without it."""
    import b200attn
    small, large = (0.02, 6e4) if dt == F16 else (0.1, 1e9)
    f = Filled(1, 2, D, 16, bits, dt, [512], seed=207)
    q = (0.5 + 0.3 * torch.from_numpy(ora.seeded_normal((1, 2 * G, D), 209))).to(dt).cuda()
    k, v = f.k[0].clone(), (f.v[0].float() * small).to(dt)
    k[0, :, at] = -160 / D ** 0.5                            # a score of about -80
    v[0, :, at] = torch.linspace(-large, large, D).to(dt).cuda()
    with_values(f, v, k)
    for splits in (None, 1, 2, 5):
        O, L = b200attn.decode_paged_quant(q, f.cache, f.btg, f.kl, splits=splits)
        check_own_steps(f, q, O, L)
    assert b200attn.device_error_flags() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("D,bits,dt,G", RANGE, ids=str)
@pytest.mark.parametrize("rise", [60.0, -60.0])
def test_values_shrink_while_scores_rise(D, bits, dt, G, rise):
    """Scores that rise by 60 along the sequence while the values shrink, and the other way round:
    what counts at the end are the tokens of high score, however small their values are."""
    import b200attn
    n = 640
    f = Filled(1, 2, D, 32, bits, dt, [n], seed=217)
    q = (0.5 + 0.3 * torch.from_numpy(ora.seeded_normal((1, 2 * G, D), 219))).to(dt).cuda()
    ramp = torch.linspace(0, 1, n)[None, None, :, None].cuda()
    k = (0.2 * f.k[0].float() + 2 * rise * ramp / D ** 0.5).to(dt)
    fall = ramp if rise > 0 else 1 - ramp
    v = (f.v[0].float() * (3e3 * 10.0 ** (-6 * fall) if dt == F16 else 10.0 ** (9 - 18 * fall))).to(dt)
    with_values(f, v, k)
    for splits in (None, 1, 3):
        O, L = b200attn.decode_paged_quant(q, f.cache, f.btg, f.kl, splits=splits)
        check_own_steps(f, q, O, L)


@pytest.mark.gpu
@pytest.mark.parametrize("bits,dt,G", [(4, F16, 4), (8, F16, 8), (4, BF16, 8), (8, BF16, 3)], ids=str)
@pytest.mark.parametrize("which", [0, 1])
def test_channel_groups_of_unequal_size(bits, dt, G, which):
    """One group of 64 channels whose values are a small part of the other's."""
    import b200attn
    f = Filled(1, 2, 128, 16, bits, dt, [700], seed=227)
    q = torch.from_numpy(ora.seeded_normal((1, 2 * G, 128), 229)).to(dt).cuda()
    size = torch.full((128,), 1e4 if dt == F16 else 1e3)
    size[64 * which:64 * which + 64] = 1e-2 if dt == F16 else 1e-9
    with_values(f, (f.v[0].float() * size.cuda()).to(dt))
    for splits in (None, 1, 4):
        O, L = b200attn.decode_paged_quant(q, f.cache, f.btg, f.kl, splits=splits)
        check_own_steps(f, q, O, L)


@pytest.mark.gpu
def test_values_of_zero_before_others():
    """Tokens whose groups have no step at all while the scores rise, then tokens that have one."""
    import b200attn
    for dt, bits in ((F16, 4), (BF16, 8)):
        f = Filled(1, 1, 64, 16, bits, dt, [512], seed=237)
        q = (0.5 + 0.3 * torch.from_numpy(ora.seeded_normal((1, 4, 64), 239))).to(dt).cuda()
        ramp = torch.linspace(0, 1, 512)[None, None, :, None].cuda()
        k = (0.2 * f.k[0].float() + 2 * 200 * ramp / 8).to(dt)
        v = f.v[0].clone()
        v[:, :, :500] = 0
        with_values(f, v, k)
        for splits in (1, 2):
            O, L = b200attn.decode_paged_quant(q, f.cache, f.btg, f.kl, splits=splits)
            check_own_steps(f, q, O, L)


@pytest.mark.gpu
@pytest.mark.parametrize("Hkv,page", [(16, 16), (32, 16), (3, 64)])
def test_read_back_with_a_loose_bound(Hkv, page):
    """max_len only has to bound the lengths: 2^31 - 1 reads what the longest length reads."""
    import b200attn
    lens = [40, 0, 7]
    f = Filled(3, Hkv, 64, page, 4, F16, lens, seed=247)
    cu = torch.tensor([0, 40, 40, 47], dtype=torch.int32, device="cuda")
    want = b200attn.read_paged_quant(f.cache, f.btg, cu, 47, 40)
    got = b200attn.read_paged_quant(f.cache, f.btg, cu, 47, 2 ** 31 - 1)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    start = torch.tensor([39, 0, 5], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 1, 1, 3], dtype=torch.int32, device="cuda")
    got = b200attn.read_paged_quant(f.cache, f.btg, cu, 3, 2 ** 31 - 1, start=start)
    for a, w in zip(got, want):
        assert torch.equal(a, w[[39, 45, 46]])
    assert b200attn.device_error_flags() == 0


def test_numbers_past_32_bits_are_refused():
    """No argument reaches the library without its upper bits, through either binding."""
    from b200attn import quantcache as qc
    big = (1 << 32) + 16
    with pytest.raises(RuntimeError, match="32 bits"):
        qc.block_bytes((1 << 32) + 128, 16, 4)
    with pytest.raises(RuntimeError, match="32 bits"):
        qc._plan(1, 8, 8, 128, 4, 100, 1 << 29)
    # places of the ints among the arguments
    calls = {"_append": (24, range(7, 17)), "_read": (17, range(6, 16)),
             "_select": (19, range(7, 16)), "_decode": (23, [5, *range(9, 19)])}
    for name, (n, ints) in calls.items():
        for f in {getattr(qc, name), getattr(qc, name + "_ct")}:
            for i in range(n):
                for value in (big, -big):
                    args = [0] * n
                    args[i] = value
                    if name == "_decode" and i == 22:
                        continue                     # the scale
                    if i in ints:
                        with pytest.raises(RuntimeError, match="32 bits"):
                            f(*args)
                    else:
                        assert f(*args) != 0         # refused by the library: no device, or no such shape


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 200])
def test_lengths_that_do_not_advance(T):
    """A negative length stays what it is, for one token and for many (which take two ways to the
    lengths); one next to 2^31 stops there.  Their tokens are dropped, the others' are not."""
    import b200attn
    cache = b200attn.QuantCache.empty(16, 16, 3, 64, dtype=F16)
    bt = torch.full((4, 14), -1, dtype=torch.int32, device="cuda")
    bt[1] = torch.arange(14)
    top = 2 ** 31 - 1
    kl = torch.tensor([-4, 3, top - T + 1, -2 ** 31], dtype=torch.int32, device="cuda")
    k = torch.ones(4, 3, T, 64, dtype=F16, device="cuda")
    b200attn.device_error_flags()
    b200attn.append_paged_quant(k, k, cache, bt, kl)
    assert kl.tolist() == [-4, 3 + T, top, -2 ** 31]
    assert b200attn.device_error_flags() == 4
    got = cache.params(0)[:14, 0, :, 0, 1].flatten()
    assert (got[3:3 + T] == 1).all() and not got[:3].any() and not got[3 + T:].any()


def test_kernels_promise_no_constant_memory():
    """Kernels that may start before the one ahead has ended (griddepcontrol) must not declare
    what that one writes as constant while they live: `const T* __restrict__`."""
    import os
    import re
    from conftest import PKG_PARENT
    for name in ("kvquant.cuh", "kvquant_sm100.cu", "kvquant_decode_sm100.cu"):
        text = open(os.path.join(PKG_PARENT, "csrc", name)).read()
        assert "pdl_wait" in text
        assert not re.findall(r"const\s+\w+\s*\*\s*(?:const\s+)?__restrict__", text), name
        assert "__ldg(" not in text and "ld.global.nc" not in text


def test_a_warp_agrees_on_its_waits():
    """A bounded wait may run out in some lanes of a warp only; what the warp does next has
    shuffles, so the lanes' answers are made one by a vote.  (Read from the source: no test can
    place a copy's arrival between two lanes' looks.)"""
    import os
    import re
    from conftest import PKG_PARENT
    text = open(os.path.join(PKG_PARENT, "csrc", "kvquant_decode_sm100.cu")).read()
    waits = re.findall(r"^.*\bmbar_wait\(.*$", text, re.M)
    assert waits and all("__all_sync(0xffffffffu," in w for w in waits)


def test_pool_takes_any_iterable_of_sequences():
    """A generator is as good as a list; one sequence under two names is one sequence."""
    from b200attn.quantcache import QuantPagePool
    pool = QuantPagePool(10, 16, 2, 64, max_seqs=3, max_pages=8, device="cpu")
    wrote = []
    pool._write = lambda k, v, bt, lens: (wrote.append(k.shape[0]), lens.add_(k.shape[2]))
    k = torch.zeros(2, 2, 5, 64, dtype=F16)
    pool.append(k, k, seqs=(s for s in (2, 0)))
    pool.append(k, k, seqs=torch.tensor([1, 2]))
    pool.append(k, k, seqs=[-1, 0])
    assert wrote == [2, 2, 2] and pool.lengths() == [10, 5, 15]
    for bad in ([2, -1], torch.tensor([1, 1]), iter([0, 0])):
        with pytest.raises(RuntimeError, match="once"):
            pool.append(k, k, seqs=bad)
    with pytest.raises(IndexError):
        pool.append(k, k, seqs=[0, 3])
    assert pool.lengths() == [10, 5, 15]


@pytest.mark.gpu
@pytest.mark.parametrize("D,bits,dt,G", RANGE, ids=str)
@pytest.mark.parametrize("power", [18, 26, 33, 60])
def test_scores_of_any_size(D, bits, dt, G, power):
    """Scores up to 2^60: one token's is the largest by 2 percent, and it takes all the weight."""
    import b200attn
    if dt == F16 and power == 60:
        power = 36
    n = 300
    f = Filled(1, 2, D, 16, bits, dt, [n], seed=257)
    q = torch.full((1, 2 * G, D), 2.0 ** (power // 2 - 3), dtype=dt, device="cuda")
    rows = torch.from_numpy(np.random.default_rng(5).permutation(n)) / n
    size = 0.9 - 0.4 * rows                                  # 0.5 .. 0.9 and one at 0.92
    size[211] = 0.92
    k = (size[None, None, :, None].cuda() * 2.0 ** (power - power // 2 - 3)).to(dt).expand(1, 2, n, D)
    with_values(f, k=k)
    assert float(q.max()) * float(k.max()) * D ** 0.5 > 2.0 ** (power - 4)
    for splits in (None, 1, 2):
        O, L = b200attn.decode_paged_quant(q, f.cache, f.btg, f.kl, splits=splits)
        check_own_steps(f, q, O, L)
    assert b200attn.device_error_flags() == 0


@pytest.mark.gpu
def test_tiny_queries_and_scales():
    """Queries next to the smallest of bf16 with keys next to the largest and a tiny scale: the
    factor that takes a score to log2 units is a subnormal number, and counts as it is."""
    import b200attn
    f = Filled(1, 1, 64, 16, 8, BF16, [100], seed=267)
    with_values(f, k=(f.k[0].float().abs() * 2.0 ** 124).to(BF16))  # all of one sign: sums count
    q = (torch.from_numpy(ora.seeded_normal((1, 4, 64), 269)).abs() * 2.0 ** -118).bfloat16().cuda()
    for scale in (1e-6, 1e-9, 1e-11):
        O, L = b200attn.decode_paged_quant(q, f.cache, f.btg, f.kl, scale=scale)
        check_attention(f, q, O, L, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("bits,dt,G", [(4, F16, 4), (8, F16, 8), (4, BF16, 8), (8, BF16, 3)], ids=str)
@pytest.mark.parametrize("which", [0, 1])
def test_query_groups_of_unequal_size(bits, dt, G, which):
    """One group of 64 channels whose queries are a small part of the other's, and whose keys are
    as much larger: both count for the scores."""
    import b200attn
    f = Filled(1, 2, 128, 16, bits, dt, [300], seed=277)
    part = 1e-7 if dt == F16 else 1e-12
    most = 1e3 if dt == F16 else 1e6
    size = torch.full((128,), most)
    size[64 * which:64 * which + 64] = part * most
    q = (torch.from_numpy(ora.seeded_normal((1, 2 * G, 128), 279)) * size).to(dt).cuda()
    with_values(f, k=(f.k[0].float() / size.cuda()).to(dt))
    for splits in (None, 1, 3):
        O, L = b200attn.decode_paged_quant(q, f.cache, f.btg, f.kl, splits=splits)
        check_own_steps(f, q, O, L)


def test_scratch_and_warps_follow_the_kernels():
    """Sizes that the host asks the library for, at the bounds where they change."""
    from b200attn import _lib
    from b200attn import quantcache as qc
    lib = _lib.load()
    assert lib.b2a_kvq_select_keys_words(3, 8, 2048) == 0 == qc._keys_words(3, 8, 2048)
    assert lib.b2a_kvq_select_keys_words(3, 8, 2049) == 3 * 8 * 2049 == qc._keys_words(3, 8, 2049)
    assert lib.b2a_kvq_select_keys_words(65535, 8, 1 << 20) == 65535 * 8 << 20
    assert lib.b2a_kvq_select_keys_words(0, 8, 4096) == 0
    for D, bits, warps in ((128, 4, 12), (128, 8, 6), (64, 4, 16), (64, 8, 12)):
        assert lib.b2a_kvq_decode_workers(64, 8, D, bits, 1 << 20) == 148 * warps


@pytest.mark.gpu
def test_captured_fork_and_join():
    """A capture that forks: two caches' steps on two streams that meet in one decode each, and
    a second join over both; replays give what the same calls give eagerly."""
    import b200attn
    B, H, Hkv, D = 2, 8, 2, 64
    fs = [Filled(B, Hkv, D, 16, 4, F16, [300, 90], seed=287 + i, index=True, width=24) for i in (0, 1)]
    x = torch.from_numpy(ora.seeded_normal((B, Hkv, 1, D), 289)).half().cuda()
    q = torch.from_numpy(ora.seeded_normal((B, H, D), 290)).half().cuda()
    at = fs[0].kl - 1
    side = torch.cuda.Stream()

    def step():
        main = torch.cuda.current_stream()
        b200attn.append_paged_quant(x, x, fs[0].cache, fs[0].btg, at, advance=False)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            b200attn.append_paged_quant(x, x, fs[1].cache, fs[1].btg, at, advance=False)
            pages = b200attn.select_pages(q, fs[1].cache, fs[1].btg, fs[1].kl, 5)
        first = b200attn.decode_paged_quant(q, fs[0].cache, fs[0].btg, fs[0].kl)
        main.wait_stream(side)
        return first + b200attn.decode_paged_quant(q, fs[1].cache, fs[1].btg, fs[1].kl, pages=pages) + [pages]

    warm = torch.cuda.Stream()
    with torch.cuda.stream(warm):
        step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for it in range(3):
        x.copy_(torch.from_numpy(ora.seeded_normal((B, Hkv, 1, D), 291 + it)).half())
        q.copy_(torch.from_numpy(ora.seeded_normal((B, H, D), 295 + it)).half())
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        for a, w in zip(got, step()):
            torch.cuda.synchronize()
            assert torch.equal(a, w)
        for f in fs:
            for b in range(B):
                f.k[b][0, :, -1] = f.v[b][0, :, -1] = x[b, :, 0]
        check_attention(fs[0], q, got[0], got[1])
        check_attention(fs[1], q, got[2], got[3], pages=got[4].cpu().numpy())
    assert b200attn.device_error_flags() == 0


@pytest.mark.gpu
def test_shared_pages_and_repeated_entries():
    """Sequences that share the pages of a common beginning; a page that a list names twice."""
    import b200attn
    f = Filled(1, 2, 128, 16, 8, BF16, [64 + 21], seed=307)
    extra = b200attn.QuantCache.empty(8, 16, 2, 128, bits=8, dtype=BF16)
    extra.data[:f.cache.num_pages - 2] = f.cache.data[f.btg[0].long()]   # in order: 0 .. 5
    bt = torch.tensor([[0, 1, 2, 3, 4, 5], [0, 1, 2, 3, 6, 7]], dtype=torch.int32, device="cuda")
    kl = torch.tensor([85, 64], dtype=torch.int32, device="cuda")
    k, v = (torch.from_numpy(ora.seeded_normal((1, 2, 21, 128), s)).bfloat16().cuda() for s in (308, 309))
    b200attn.append_paged_quant(k, v, extra, bt[1:], kl[1:])
    assert kl.tolist() == [85, 85]
    q = torch.from_numpy(ora.seeded_normal((2, 4, 128), 310)).bfloat16().cuda()
    both = Filled.__new__(Filled)
    both.cache, both.lens, both.page, both.bits, both.dt, both.name = extra, [85, 85], 16, 8, BF16, "bfloat16"
    both.k = [f.k[0], torch.cat((f.k[0][:, :, :64], k), 2)]
    both.v = [f.v[0], torch.cat((f.v[0][:, :, :64], v), 2)]
    O, L = b200attn.decode_paged_quant(q, extra, bt, kl)
    check_attention(both, q, O, L)
    lists = np.array([[[2, 2, 5, 0], [1, 4, 1, 1]], [[5, 5, 5, 5], [-1, 3, 3, 9]]], np.int32)
    for splits in (None, 1, 3):
        O, L = b200attn.decode_paged_quant(q, extra, bt, kl, pages=torch.from_numpy(lists).cuda(),
                                           splits=splits)
        check_attention(both, q, O, L, pages=lists)
    assert b200attn.device_error_flags() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("splits", [1, 7])
def test_decode_without_lse(splits):
    """The C entry with lse == NULL gives the same O."""
    import ctypes
    import b200attn
    from b200attn import _lib
    f = Filled(3, 2, 64, 16, 4, F16, [0, 300, 33], seed=317)
    q = torch.from_numpy(ora.seeded_normal((3, 6, 64), 319)).half().cuda()
    want = b200attn.decode_paged_quant(q, f.cache, f.btg, f.kl, splits=splits)
    lib = _lib.load()
    workers = splits * 6
    ws = torch.empty(lib.b2a_kvq_decode_workspace_floats(3, 6, 2, 64, workers), device="cuda")
    O = torch.empty_like(q)
    strides = (ctypes.c_int64 * 2)(6 * 64, 64)
    _lib.check(lib.b2a_kvq_decode_paged(
        q.data_ptr(), strides, f.cache.data.data_ptr(), f.btg.data_ptr(), f.kl.data_ptr(), None, 0,
        ws.data_ptr(), O.data_ptr(), None, 3, 6, 2, 64, 16, f.btg.shape[1], f.cache.num_pages, workers,
        4, 0, 0.125, torch.cuda.current_stream().cuda_stream))
    assert torch.equal(O, want[0])


@pytest.mark.gpu
@pytest.mark.parametrize("D,bits,dt,G", RANGE, ids=str)
@pytest.mark.parametrize("n", [3, 70, 3000])
def test_values_next_to_the_largest(D, bits, dt, G, n):
    """Values up to the type's largest: their weighted mean is finite, whatever the sums of their
    products with unnormalised weights are."""
    import b200attn
    big = torch.finfo(dt).max
    f = Filled(1, 2, D, 16, bits, dt, [n], seed=327)
    g = torch.Generator().manual_seed(n)
    v = (1 - 0.3 * torch.rand(1, 2, n, D, generator=g)) * big
    v[..., 1::3] *= -1
    v[:, :, 0, 0] = big
    with_values(f, v=v.to(dt).cuda(), k=f.k[0] * 0.1)       # weights all alike
    q = torch.from_numpy(ora.seeded_normal((1, 2 * G, D), 329)).to(dt).cuda()
    for splits in (None, 1, 7):
        O, L = b200attn.decode_paged_quant(q, f.cache, f.btg, f.kl, splits=splits)
        assert torch.isfinite(O).all()
        check_own_steps(f, q, O, L)


@pytest.mark.gpu
@pytest.mark.parametrize("bits,G", [(4, 4), (8, 8)])
def test_values_next_to_the_smallest_steps(bits, G):
    """Values whose steps are next to 2^-100, the smallest that are kept, and zeros among them;
    scores of one size, and some that rise and fall by 40."""
    import b200attn
    for power, rise in ((-80, 0), (-92, 0), (-97, 0), (-80, 40), (-92, 40), (-92, -40), (-97, 40),
                        (-101, 0), (-101, 40), (-101, -40)):
        f = Filled(1, 1, 128, 16, bits, BF16, [400], seed=337)
        v = f.v[0].float() * 2.0 ** (power + bits)
        v[:, :, 100:140] = 0
        v[:, :, :, 64:] *= 2.0 ** -4
        q = torch.from_numpy(ora.seeded_normal((1, G, 128), 339))
        q = (q if rise == 0 else 0.5 + 0.3 * q).bfloat16().cuda()
        ramp = torch.linspace(0, 1, 400)[None, None, :, None].cuda() * 2 * rise / 128 ** 0.5
        with_values(f, v=v.to(BF16), k=(f.k[0].float() * (0.2 if rise else 1) + ramp).to(BF16))
        for splits in (None, 1, 5):
            O, L = b200attn.decode_paged_quant(q, f.cache, f.btg, f.kl, splits=splits)
            check_own_steps(f, q, O, L)


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(6))
def test_values_spread_over_the_range(seed):
    """Values whose size differs from token to token by up to 10^70 (bf16) or 10^8 (fp16), up to
    the type's largest: whatever counts at a head's end is there."""
    import b200attn
    rng = np.random.default_rng(seed)
    D, bits, dt, G = RANGE[seed]
    n = 900
    f = Filled(1, 2, D, 64, bits, dt, [n], seed=347 + seed)
    ten = rng.uniform(-38, 38, (1, 2, n, 1)) if dt == BF16 else rng.uniform(-4, 4.5, (1, 2, n, 1))
    if seed & 1:                                   # most of them small, a few at the upper end
        ten = np.where(rng.random(ten.shape) < 0.02, ten, ten.min() / 2)
    big = torch.finfo(dt).max
    v = f.v[0].double() * 10.0 ** torch.from_numpy(ten).cuda()
    with_values(f, v=v.clamp(-big, big).to(dt))
    q = torch.from_numpy(ora.seeded_normal((1, 2 * G, D), 349)).to(dt).cuda()
    for splits in (None, 1, 4):
        O, L = b200attn.decode_paged_quant(q, f.cache, f.btg, f.kl, splits=splits)
        check_own_steps(f, q, O, L)


@pytest.mark.gpu
def test_too_few_workers_for_the_table():
    """A worker counts its steps in 32 bits: a call that could pass that is refused."""
    from b200attn import _lib
    from b200attn import quantcache as qc
    # q data table lens pages | n_pages | workspace o lse | B H Hkv D page max_pages num_pages workers bits dtype
    args = [0] * 5 + [0] + [0] * 3 + [65535, 64, 8, 64, 64, 1 << 24, 100, 1, 4, 0, 0, 64, 64, 0.125]
    for f in (qc._decode, qc._decode_ct):
        with pytest.raises(RuntimeError, match="too few workers"):
            _lib.check(f(*args))
        args[16] = 65535 * 8
        with pytest.raises(RuntimeError, match="q must not be null"):
            _lib.check(f(*args))
        args[16] = 1


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 8])
def test_scores_creep_up_while_values_shrink(bits):
    """The maximum rises by less than one at every step and the values shrink by as much or more:
    what o holds and what its products are scaled by stay together over many small changes."""
    import b200attn
    n = 64 * 120
    f = Filled(1, 1, 64, 64, bits, BF16, [n], seed=357)
    q = torch.ones(1, 4, 64, dtype=BF16, device="cuda")
    rise = torch.arange(n).float()[None, None, :, None].cuda() / 64 * 0.4     # in all 48
    k = (0.05 * f.k[0].float() + rise / 8).to(BF16)
    for fall in (0.4, 1.2):
        with_values(f, v=(f.v[0].float() * torch.exp(30 - rise * fall / 0.4 * 0.8)).to(BF16), k=k)
        for splits in (1, 2, 9):
            O, L = b200attn.decode_paged_quant(q, f.cache, f.btg, f.kl, splits=splits)
            check_own_steps(f, q, O, L)


@pytest.mark.gpu
def test_the_heaviest_token_is_not_rounded():
    """fp16 outputs' mean square error is that of one rounding of O and one of each product p *
    step but the heaviest token's, which is its step times a power of two.

    A rounding to a spacing h has mean square h^2 / 12.  For O the spacing is known,
    2^(floor(log2 |O|) - 10).  A product x in [2^e, 2^(e+1)) has h = 2^(e - 10), and its mantissa,
    that of an exponential, is spread evenly over its logarithm: the mean of (2^e / x)^2 is
    (3 / 8) / ln 2 and the mean square 2^-20 / 12 * 0.541 of x^2.  Over 2^16 outputs, of which the
    64 channels of a head share their products' errors, the sum is within some percent of that."""
    import b200attn
    f = Filled(8, 4, 128, 16, 8, F16, [4000] * 8, seed=367)
    q = torch.from_numpy(ora.seeded_normal((8, 16, 128), 369) * 3).half().cuda()
    O, L = b200attn.decode_paged_quant(q, f.cache, f.btg, f.kl)
    got = result = products = 0.0
    for b in range(8):
        K, V = (f.codes(b, s) for s in (0, 1))
        for h in range(4):
            k, v = oq.values(*(x[h] for x in K)), oq.values(*(x[h] for x in V))
            Or, Lr = oq.attend(np_of(q)[b, 4 * h:4 * h + 4], k, v, 128 ** -0.5)
            s = np_of(q)[b, 4 * h:4 * h + 4].astype(np.float64) @ k.T * 128 ** -0.5
            p = np.exp(s - Lr[:, None])
            p[np.arange(4), p.argmax(-1)] = 0
            off = np.repeat(V[1][h].astype(np.float64), 64, -1) * (V[0][h] - 128.0)
            got += ((np_of(O)[b, 4 * h:4 * h + 4] - Or) ** 2).sum()
            result += (2.0 ** (2 * np.floor(np.log2(np.abs(Or))) - 20) / 12).sum()
            products += (p ** 2 @ off ** 2).sum() * 2.0 ** -20 / 12 * 0.375 / np.log(2)
    assert got <= 1.04 * (result + products), (got, result, products)
