"""Operators of the quantised paged KV cache: their cases, plain forms and exact values.

A cache holds keys and values in 4 or 8 bits.  The block of one (page, KV head)
is [K codes | V codes | K params | V params]: codes are token-major rows of
D*bits/8 bytes (low nibble first), params one (scale, min) pair in the cache's
dtype per token and group of 64 channels; a code c stands for scale*c + min.
An optional index holds, per (page, KV head), the channel minima and maxima of
the page's keys in int8 with one fp32 scale; a query scores pages with it.

kinds: "write"  append new tokens, then read just those back
       "read"   read whole histories back, packed token-major
       "decode" attention of one query token over the whole cache
       "sparse" append one token (with the index), select pages, attend to those
"""
import math
import os
import sys

import torch

own = False

DT = {"fp16": torch.float16, "bf16": torch.bfloat16}
GROUP = 64
TINY = 2.0 ** -100


# ------------------------------------------------------------------- cases
def listed():
    return [
        # one decode step's new token of every sequence of a serving batch
        dict(name="write_4bit_token", kind="write", B=64, Hkv=8, G=4, D=128, page=16, bits=4, dtype="fp16", T=1, lo=512, hi=4096),
        # a prompt chunk, starting inside a page for some sequences
        dict(name="write_4bit_prompt", kind="write", B=4, Hkv=8, G=4, D=128, page=16, bits=4, dtype="bf16", T=8192, lo=0, hi=100),
        # an odd chunk of a smaller model, 8 bits
        dict(name="write_8bit_odd", kind="write", B=3, Hkv=4, G=2, D=64, page=32, bits=8, dtype="fp16", T=1777, lo=1, hi=999),
        # a cached prefix of every sequence, read back for a chunk of prefill over it
        dict(name="read_4bit_history", kind="read", B=16, Hkv=8, G=4, D=128, page=16, bits=4, dtype="fp16", lo=512, hi=16384),
        # short ragged prefixes, 8 bits
        dict(name="read_8bit_short", kind="read", B=7, Hkv=4, G=2, D=64, page=64, bits=8, dtype="bf16", lo=1, hi=700),
        # one short chat: latency
        dict(name="decode_4bit_one", kind="decode", B=1, Hkv=8, G=4, D=128, page=16, bits=4, dtype="fp16", lo=777, hi=777),
        # a serving batch of ragged lengths in 16-token pages
        dict(name="decode_4bit_batch", kind="decode", B=64, Hkv=8, G=4, D=128, page=16, bits=4, dtype="fp16", lo=512, hi=32768),
        # one long context
        dict(name="decode_4bit_long", kind="decode", B=1, Hkv=8, G=4, D=128, page=32, bits=4, dtype="bf16", lo=131072, hi=131072),
        # heads that share nothing, 8 bits, D = 64
        dict(name="decode_8bit_batch", kind="decode", B=32, Hkv=8, G=1, D=64, page=64, bits=8, dtype="bf16", lo=100, hi=8192),
        # long contexts of which a query reads 2048 tokens
        dict(name="sparse_4bit_long", kind="sparse", B=2, Hkv=8, G=4, D=128, page=16, bits=4, dtype="bf16", top=128, lo=130000, hi=131000),
        # a serving batch with 1024 tokens a query
        dict(name="sparse_4bit_batch", kind="sparse", B=32, Hkv=8, G=4, D=128, page=16, bits=4, dtype="fp16", top=64, lo=512, hi=16384),
        # few short sequences, some with fewer pages than are asked for
        dict(name="sparse_8bit_short", kind="sparse", B=5, Hkv=2, G=8, D=64, page=32, bits=8, dtype="fp16", top=24, lo=1, hi=3000),
    ]


def draw(rng):
    def log(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    kind = rng.choice(["write", "read", "decode", "sparse"])
    c = dict(kind=kind, B=log(1, 64), Hkv=rng.choice([1, 2, 4, 5, 8]), G=rng.randint(1, 8), D=rng.choice([64, 128]),
             page=rng.choice([16, 32, 64]), bits=rng.choice([4, 4, 8]), dtype=rng.choice(["fp16", "bf16"]))
    most = {"write": 32768, "read": 131072, "decode": 524288, "sparse": 262144}[kind]  # tokens of all sequences
    if kind == "write":
        c["T"] = log(1, max(1, most // c["B"]))
        c["lo"], c["hi"] = 0, log(1, 4096)
    else:
        c["hi"] = log(1, min(131071, most // c["B"]))
        c["lo"] = rng.randint(0 if kind == "decode" else 1, c["hi"])
    if kind == "sparse":
        c["top"] = log(1, max(1, min(200, most // (c["B"] * c["page"]))))
    return c


# ------------------------------------------------------------------- inputs
def lengths(case, gen):
    """Cached lengths, one per sequence, as a list (known to the program, which allocates the pages)."""
    n = torch.randint(case["lo"], case["hi"] + 1, (case["B"],), generator=gen).tolist()
    return [case["hi"] if case["lo"] == case["hi"] else v for v in n]


def prepare(case, seed):
    B, Hkv, G, D, page, bits = (case[k] for k in ("B", "Hkv", "G", "D", "page", "bits"))
    dt, H = DT[case["dtype"]], case["Hkv"] * case["G"]
    host = torch.Generator().manual_seed(seed)
    gen = torch.Generator("cuda").manual_seed(seed)
    T = {"write": case.get("T"), "sparse": 1}.get(case["kind"], 0)
    # the lengths of a "read" are the case's own: its outputs' sizes go by their sum
    lens = lengths(case, torch.Generator().manual_seed(case["hi"]) if case["kind"] == "read" else host)
    pages = [-(-(n + T) // page) for n in lens]
    P = sum(pages) + 2
    perm = torch.randperm(P, generator=host)
    table = torch.full((B, max(max(pages), 1)), -1, dtype=torch.int32)
    at = 0
    for b in range(B):
        table[b, :pages[b]] = perm[at:at + pages[b]].int()
        at += pages[b]
    st = dict(case=case, shape=(page, D, bits, dt), table=table.cuda(), lens=torch.tensor(lens, dtype=torch.int32, device="cuda"))

    # keys have a few channels with a large mean, as learned ones do; pages differ in where they lie
    mean = torch.randn(Hkv, 1, D, generator=gen, device="cuda")
    mean = torch.where(mean.abs() > 2, mean * 2, mean * 0.3)

    def new_kv(n, t):
        k = torch.randn(n, Hkv, t, D, generator=gen, device="cuda") + 0.5 * torch.randn(n, Hkv, 1, D, generator=gen, device="cuda") + mean
        return k.to(dt), torch.randn(n, Hkv, t, D, generator=gen, device="cuda").to(dt)

    st["data"] = torch.empty(P, Hkv, 2 * page * (D * bits // 8 + D // GROUP * 4), dtype=torch.uint8, device="cuda")
    sparse = case["kind"] == "sparse"
    st["index"] = torch.zeros(P, Hkv, 2, D, dtype=torch.int8, device="cuda") if sparse else None
    st["index_scale"] = torch.zeros(P, Hkv, device="cuda") if sparse else None
    step = max(1, (1 << 26) // (Hkv * page * D))
    for p in range(0, P, step):
        n = min(step, P - p)
        for side, x in enumerate(new_kv(n, page)):
            codes, par = quantise(x, bits)
            block_codes(st["data"], st["shape"], side)[p:p + n] = codes
            block_params(st["data"], st["shape"], side)[p:p + n] = par
            if sparse and side == 0:
                st["index"][p:p + n], st["index_scale"][p:p + n] = bounds(dequantise(codes, par, bits).to(dt).float(), None)
    if T:
        # [B, T, Hkv, D] from a projection, seen as [B, Hkv, T, D]
        st["k_new"], st["v_new"] = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in new_kv(B, T))
    if case["kind"] in ("write", "read"):
        n = [T] * B if T else lens
        st["start"] = st["lens"] if T else None
        st["total"], st["longest"] = sum(n), max(n)
        st["cu"] = torch.tensor([0] + n, device="cuda").cumsum(0).int()
    else:
        st["q"] = torch.randn(B, H, D, generator=gen, device="cuda").to(dt)
        st["kv_lens"] = st["lens"] + T
    return st


# ------------------------------------------------------------------- plain forms
def block_codes(data, shape, side):
    """K (side 0) or V (1) codes as a view [..., page, D*bits/8]."""
    page, D, bits, _ = shape
    n = page * (D * bits // 8)
    return data[..., side * n:(side + 1) * n].unflatten(-1, (page, D * bits // 8))


def block_params(data, shape, side):
    """K or V params as a view [..., page, D/64, 2] of the cache's dtype."""
    page, D, bits, dt = shape
    at, n = 2 * page * (D * bits // 8), page * (D // GROUP) * 4
    return data[..., at + side * n:at + (side + 1) * n].view(dt).unflatten(-1, (page, D // GROUP, 2))


def quantise(x, bits):
    """Codes (packed bytes [..., D*bits/8]) and params [..., D/64, 2] of x [..., D]."""
    n, dt = 2 ** bits - 1, x.dtype
    g = x.unflatten(-1, (-1, GROUP)).float()
    low = g.amin(-1, keepdim=True)
    exact = (g.amax(-1, keepdim=True) * 0.5 - low * 0.5) * (2 / n)
    near = exact.to(dt)
    bits_of = near.view(torch.int16)
    up = torch.where(near.float() < exact, bits_of + 1, bits_of).view(dt)
    down = torch.where(near.float() > exact, bits_of - 1, bits_of).view(dt)
    scale = torch.where((low + n * up.float()).to(dt).isinf(), down, up).float()
    scale = torch.where(scale < TINY, 0.0, scale)
    code = ((g * 0.5 - low * 0.5) * (scale * 0.5).reciprocal()).round().clamp(0, n)
    code = torch.where(scale == 0, 0.0, code)
    bad = ~g.isfinite().all(-1, keepdim=True)
    code = torch.where(bad, 0.0, code).to(torch.uint8).flatten(-2)
    par = torch.where(bad, float("nan"), torch.cat((scale, low), -1)).to(dt)
    return (code[..., ::2] | code[..., 1::2] << 4 if bits == 4 else code), par


def dequantise(codes, par, bits):
    """The values in 32 bits, not rounded to the cache's dtype."""
    if bits == 4:
        codes = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    par = par.float()
    return (codes.unflatten(-1, (-1, GROUP)).float() * par[..., :1] + par[..., 1:]).flatten(-2)


def bounds(k, valid):
    """Index codes [..., 2, D] and scale [...] of keys k [..., tokens, D]; valid [..., tokens, 1] or None."""
    if valid is None:
        both = torch.stack((k.amin(-2), k.amax(-2)), -2)
    else:
        both = torch.stack((k.masked_fill(~valid, math.inf).amin(-2), k.masked_fill(~valid, -math.inf).amax(-2)), -2)
    code, scale = signed8(both, (-2, -1))
    return code.to(torch.int8), scale[..., 0, 0]


def signed8(x, dims):
    """x over dims in whole numbers of -127..127 (as floats) and the scale; a NaN or infinity: zeros and NaN."""
    top = x.abs().amax(dims, keepdim=True)
    ok = top.isfinite()
    scale = torch.where(ok, top * (1 / 127), float("nan"))
    return torch.where(scale >= TINY, (x * scale.reciprocal()).round().clamp(-127, 127), 0.0), scale


def attend(q, k, v, valid):
    """[O, L] of q [B, Hkv, G, D] over k, v [B, Hkv, N, D] where valid [B, Hkv or 1, 1, N]."""
    s = (q.float() @ k.transpose(-1, -2) * q.shape[-1] ** -0.5).masked_fill(~valid, -math.inf)
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = (s - top).exp()
    total = p.sum(-1, keepdim=True)
    o = p @ v.masked_fill(~valid.transpose(-1, -2), 0.0) / torch.where(total == 0, 1.0, total)
    return [o.to(q.dtype).flatten(1, 2), (top + total.log())[..., 0].flatten(1, 2)]


def page_values(st, table, heads, side):
    """Read-back values of the pages in table (of the given heads, or of all: None) in 32 bits."""
    shape = st["shape"]
    at = table.long().clamp(min=0)
    at = at if heads is None else (at, heads)
    return dequantise(block_codes(st["data"], shape, side)[at], block_params(st["data"], shape, side)[at], shape[2])


def plain_append(st):
    page, D, bits, dt = st["shape"]
    B, Hkv, T, _ = st["k_new"].shape
    pos = st["lens"][:, None].long() + torch.arange(T, device="cuda")
    to, slot = st["table"].long().gather(1, pos // page), pos % page
    for side, x in ((0, st["k_new"]), (1, st["v_new"])):
        codes, par = quantise(x.transpose(1, 2), bits)
        block_codes(st["data"], st["shape"], side)[to, :, slot] = codes
        block_params(st["data"], st["shape"], side)[to, :, slot] = par
    if st["index"] is not None:
        first = st["lens"].long() // page
        touched = first[:, None] + torch.arange((T - 1) // page + 2, device="cuda")
        live = touched * page < (st["lens"] + T)[:, None]
        touched = torch.where(live, touched, first[:, None])  # twice the same page writes the same twice
        at = st["table"].long().gather(1, touched)
        token = touched[..., None] * page + torch.arange(page, device="cuda")
        valid = (token < (st["lens"] + T)[:, None, None])[:, :, None, :, None]
        code, scale = bounds(page_values(st, at, None, 0).to(dt).float(), valid)
        st["index"][at], st["index_scale"][at] = code, scale


def plain_read(st):
    page, D, bits, dt = st["shape"]
    cu = st["cu"].long()
    row = torch.arange(st["total"], device="cuda")
    b = torch.searchsorted(cu, row, right=True) - 1
    pos = row - cu[b] + (0 if st["start"] is None else st["start"].long()[b])
    at, slot = st["table"].long()[b, pos // page], pos % page
    return [dequantise(block_codes(st["data"], st["shape"], s)[at, :, slot], block_params(st["data"], st["shape"], s)[at, :, slot], bits).to(dt)
            for s in (0, 1)]


def plain_decode(st):
    page, D, bits, dt = st["shape"]
    B, MP = st["table"].shape
    Hkv = st["data"].shape[1]
    k, v = (page_values(st, st["table"], None, s).transpose(1, 2).flatten(2, 3) for s in (0, 1))
    valid = torch.arange(MP * page, device="cuda") < st["kv_lens"][:, None, None, None]
    return attend(st["q"].unflatten(1, (Hkv, -1)), k, v, valid)


def plain_select(st):
    """Pages [B, Hkv, top] (logical numbers, ascending, -1 behind the last)."""
    page = st["shape"][0]
    Hkv, top_k = st["data"].shape[1], st["case"]["top"]
    q = st["q"].unflatten(1, (Hkv, -1)).float()
    q8, scale = signed8(q, (-1,))
    at = st["table"].long().clamp(min=0)
    index = st["index"][at].float()  # [B, MP, Hkv, 2, D]
    low, high = (index[:, :, :, i].permute(0, 2, 3, 1) for i in (0, 1))
    dot = q8.clamp(max=0) @ low + q8.clamp(min=0) @ high  # whole numbers below 2^24: exact
    score = (dot * scale) * st["index_scale"][at].transpose(1, 2)[:, :, None]
    score = torch.where(score.isnan(), math.inf, score).amax(2)
    count = -(-st["kv_lens"].long() // page)[:, None, None]
    number = torch.arange(at.shape[1], device="cuda")
    score = torch.where(number == count - 1, math.inf, score)
    # behind the last page: after everything, even after scores of -infinity
    order = torch.sort(torch.where(number < count, score, -math.inf), dim=-1, descending=True, stable=True)[1]
    chosen = order[..., :top_k]
    chosen = torch.sort(torch.where(chosen < count, chosen, 1 << 30), dim=-1)[0]
    chosen = torch.nn.functional.pad(chosen, (0, top_k - chosen.shape[-1]), value=1 << 30)
    return torch.where(chosen == 1 << 30, -1, chosen).int()


def plain_sparse(st):
    plain_append(st)
    page = st["shape"][0]
    B, Hkv = st["table"].shape[0], st["data"].shape[1]
    pages = plain_select(st)
    at = st["table"].gather(1, pages.clamp(min=0).long().flatten(1)).view(pages.shape)
    heads = torch.arange(Hkv, device="cuda")[:, None]
    k, v = (page_values(st, at, heads, s).flatten(2, 3) for s in (0, 1))
    token = pages[..., None] * page + torch.arange(page, device="cuda")
    valid = ((pages[..., None] >= 0) & (token < st["kv_lens"][:, None, None, None])).flatten(2)[:, :, None]
    return attend(st["q"].unflatten(1, (Hkv, -1)), k, v, valid) + [pages]


# ------------------------------------------------------------------- one pass
def run(state):
    st, kind = state, state["case"]["kind"]
    if not own:
        if kind == "write":
            plain_append(st)
        return {"write": plain_read, "read": plain_read, "decode": plain_decode, "sparse": plain_sparse}[kind](st)
    b200attn = package()
    page, D, bits, dt = st["shape"]
    cache = b200attn.QuantCache(st["data"], page_size=page, head_dim=D, bits=bits, dtype=dt, index=st["index"], index_scale=st["index_scale"])
    if kind in ("write", "sparse"):
        b200attn.append_paged_quant(st["k_new"], st["v_new"], cache, st["table"], st["lens"], advance=False)
    if kind in ("write", "read"):
        return b200attn.read_paged_quant(cache, st["table"], st["cu"], st["total"], st["longest"], start=st["start"])
    if kind == "decode":
        return b200attn.decode_paged_quant(st["q"], cache, st["table"], st["kv_lens"])
    pages = b200attn.select_pages(st["q"], cache, st["table"], st["kv_lens"], st["case"]["top"])
    return b200attn.decode_paged_quant(st["q"], cache, st["table"], st["kv_lens"], pages=pages) + [pages]


def package():
    """The repository's package, which lies beside this folder."""
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flashattn-cuda_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import b200attn
    return b200attn


def work(case):
    """Each cached token's codes and params once; new tokens, read-back values and queries in 16 bits."""
    B, Hkv, G, D, page, bits = (case[k] for k in ("B", "Hkv", "G", "D", "page", "bits"))
    held = 2 * (D * bits // 8 + D // GROUP * 4)  # a token of one KV head, K and V
    mean = B * (case["lo"] + case["hi"]) / 2  # lengths are uniform: their expected sum
    if case["kind"] == "write":
        rows = B * case["T"] * Hkv
        return {"bytes": rows * (2 * 4 * D + 2 * held), "flops": rows * 2 * D * 8}
    if case["kind"] == "read":
        return {"bytes": mean * Hkv * (held + 4 * D), "flops": mean * Hkv * 2 * D * 2}
    ends = B * Hkv * G * (4 * D + 4)
    if case["kind"] == "decode":
        return {"bytes": mean * Hkv * held + ends, "flops": mean * Hkv * D * (4 * G + 4)}
    pages, top = mean / page + B / 2, case["top"]
    read = B * min(top * page, (case["lo"] + case["hi"]) / 2)
    return {"bytes": pages * Hkv * (2 * D + 4) + read * Hkv * held + ends + B * Hkv * (4 * D + held + 4 * top),
            "flops": pages * Hkv * G * 4 * D + read * Hkv * D * (4 * G + 4)}


# ------------------------------------------------------------------- 64 bits
def exact(case, seed):
    """The definitions in 64 bits, sequence by sequence.  Where they round to whole codes
    they say in which steps of 32 bits, and those steps are taken here too."""
    st = prepare(case, seed)
    page, D, bits, dt = st["shape"]
    Hkv, G, kind = case["Hkv"], case["G"], case["kind"]
    NG, table, lens = D // GROUP, st["table"].tolist(), st["lens"].tolist()
    row = D * bits // 8

    def values(blocks, side):
        """[n, page, D] in 64 bits of n blocks' bytes [n, block]."""
        raw = blocks[:, side * page * row:(side + 1) * page * row].reshape(-1, page, row).long()
        if bits == 4:
            full = torch.empty(raw.shape[0], page, D, dtype=torch.long, device="cuda")
            full[..., 0::2], full[..., 1::2] = raw % 16, raw // 16
            raw = full
        at = 2 * page * row + side * page * NG * 4
        par = blocks[:, at:at + page * NG * 4].contiguous().view(dt).double().reshape(-1, page, NG, 2).repeat_interleave(GROUP, 2)
        return raw.double() * par[..., 0] + par[..., 1]

    def rounded(x):
        """What x [..., D] (finite, of ordinary size) reads back as, in 64 bits."""
        n = 2 ** bits - 1
        y = x.float().reshape(*x.shape[:-1], NG, GROUP)
        low, high = y.min(-1, keepdim=True)[0], y.max(-1, keepdim=True)[0]
        want = (high - low) * (1 / n)
        step = want.to(dt).float()
        ulp = torch.ldexp(torch.full_like(step, torch.finfo(dt).eps), torch.frexp(step)[1] - 1)
        step = torch.where(step < want, step + ulp, step)
        code = ((y - low) * step.reciprocal()).round().clamp(max=n)
        code = torch.where(step > 0, code, torch.zeros_like(code))
        return (code.double() * step.double() + low.double()).reshape(x.shape)

    if kind == "write":
        return [rounded(x.transpose(1, 2).reshape(-1, Hkv, D)) for x in (st["k_new"], st["v_new"])]
    if kind == "read":
        out = [[], []]
        for b, n in enumerate(lens):
            blocks = st["data"][table[b][:-(-n // page)]]
            for side in (0, 1):
                v = values(blocks.flatten(0, 1), side).reshape(-1, Hkv, page, D)
                out[side].append(v.transpose(1, 2).reshape(-1, Hkv, D)[:n])
        return [torch.cat(x) for x in out]
    o, lse, picked = [], [], []
    for b, n in enumerate(st["kv_lens"].tolist()):
        q = st["q"][b].double().reshape(Hkv, G, D)
        count = -(-n // page)
        if n == 0:
            o.append(torch.zeros(Hkv * G, D, dtype=torch.float64, device="cuda"))
            lse.append(torch.full((Hkv * G,), -math.inf, dtype=torch.float64, device="cuda"))
            continue
        phys = torch.tensor(table[b][:count], device="cuda")
        for h in range(Hkv):
            use = torch.arange(count, device="cuda")
            if kind == "sparse":
                fresh = [rounded(x[b, h, 0]) for x in (st["k_new"], st["v_new"])]
                at, slot = phys[-1], (n - 1) % page
                last = [values(st["data"][at, h][None], s)[0] for s in (0, 1)]
                for s in (0, 1):
                    last[s][slot] = fresh[s]
                held = last[0][:slot + 1].float().to(dt).float()
                edge = torch.stack((held.min(0)[0], held.max(0)[0]))
                far = edge.abs().max()
                idx, isc = st["index"][phys, h].double(), st["index_scale"][phys, h].clone()
                idx[-1], isc[-1] = (edge * (far * (1 / 127)).reciprocal()).round().double(), far * (1 / 127)
                far = q[h].abs().max(-1, keepdim=True)[0].float()
                q8 = (q[h].float() * (far * (1 / 127)).reciprocal()).round().double()
                dot = torch.maximum(q8[:, None] * idx[:, 0], q8[:, None] * idx[:, 1]).sum(-1)
                score = (dot.float() * (far * (1 / 127)) * isc).max(0)[0]
                score[-1] = math.inf
                use = torch.argsort(score, descending=True, stable=True)[:case["top"]].sort()[0]
                pad = torch.full((case["top"],), -1, dtype=torch.int32, device="cuda")
                pad[:use.numel()] = use.int()
                picked.append(pad)
            blocks = st["data"][phys[use], h]
            k, v = values(blocks, 0), values(blocks, 1)
            if kind == "sparse":  # the newest token's page is always among them, and the last
                k[-1], v[-1] = last
            seen = (use[:, None] * page + torch.arange(page, device="cuda")).flatten() < n
            k, v = k.flatten(0, 1)[seen], v.flatten(0, 1)[seen]
            s = q[h] @ k.T * D ** -0.5
            o.append(torch.softmax(s, -1) @ v)
            lse.append(torch.logsumexp(s, -1))
    B = case["B"]
    out = [torch.cat(o).reshape(B, Hkv * G, D), torch.cat(lse).reshape(B, Hkv * G)]
    return out + ([torch.stack(picked).reshape(B, Hkv, -1)] if kind == "sparse" else [])
