"""Operators of a decoder with grouped-query attention over an 8-bit paged cache, as they are measured.

Four steps of one layer, in the order in which a serving loop runs them:

* ``norm_rope``  RMS norm of every query and key head with its gain, and the rotation by the row's position;
* ``append``     new K and V rows into the e4m3 cache, one power-of-two scale for each page and KV head, and the int8
                 centroid of each page that becomes full;
* ``attend``     ragged paged attention over that cache (single tokens, verify blocks, prompt chunks);
* ``sparse``     the blocks that a cheap centroid score selects for each row and KV head, and attention over those.

``own`` false: elementary torch operations in 32 bits (64 where 32 lose what matters).  ``own`` true: the calls a user
makes of ``hyperkernel_b200``.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
SINK, LOCAL = 1, 2  # blocks that the sparse form always reads: the first, and the row's own with the one before it


# ------------------------------------------------------------------------------------------------------------------
# Cases
# ------------------------------------------------------------------------------------------------------------------

def listed():
    return [
        # a decode step of 64 lanes: latency counts
        dict(name="norm_rope_decode", op="norm_rope", tokens=64, heads=32, kv=8, dim=128, rot=128, pairs=False, dtype="bf16"),
        # the rows of a full prefill pass
        dict(name="norm_rope_prefill", op="norm_rope", tokens=8192, heads=64, kv=8, dim=128, rot=128, pairs=False, dtype="bf16"),
        # neighbouring pairs rotated, half of each head left unrotated, an odd row count, fp16
        dict(name="norm_rope_pairs", op="norm_rope", tokens=1333, heads=24, kv=4, dim=64, rot=32, pairs=True, dtype="f16"),
        # one new row for each of 64 lanes, most of them inside a page that holds rows already
        dict(name="append_decode", op="append", lanes=64, rows_lo=1, rows_hi=1, ctx_lo=70, ctx_hi=250, kv=8, dim=128, page=64, dtype="bf16"),
        # prompt chunks of a mixed batch: whole pages, ragged ends
        dict(name="append_prefill", op="append", lanes=16, rows_lo=5, rows_hi=2048, ctx_lo=1, ctx_hi=1000, kv=8, dim=128, page=64, dtype="bf16"),
        # one short sequence, one token: latency
        dict(name="attend_one", op="attend", lanes=1, rows_lo=1, rows_hi=1, ctx_lo=777, ctx_hi=777, heads=32, kv=8, dim=128, page=64, dtype="bf16"),
        # a decode batch with contexts spread over a factor of 32
        dict(name="attend_decode", op="attend", lanes=64, rows_lo=1, rows_hi=1, ctx_lo=1024, ctx_hi=32768, heads=64, kv=8, dim=128, page=64, dtype="bf16"),
        # the verify block of one sequence of a million tokens
        dict(name="attend_verify_long", op="attend", lanes=1, rows_lo=5, rows_hi=5, ctx_lo=1048571, ctx_hi=1048571, heads=32, kv=8, dim=128, page=64, dtype="bf16"),
        # prompt chunks over what earlier chunks left in the cache
        dict(name="attend_prefill", op="attend", lanes=4, rows_lo=512, rows_hi=2048, ctx_lo=1000, ctx_hi=6000, heads=32, kv=8, dim=128, page=64, dtype="bf16"),
        # small heads, three query heads to a KV head, small pages, verify blocks of odd lengths
        dict(name="attend_odd", op="attend", lanes=13, rows_lo=1, rows_hi=7, ctx_lo=3, ctx_hi=5000, heads=12, kv=4, dim=64, page=16, dtype="f16"),
        # 64 blocks of 64 tokens out of up to 2048 for each lane's next token
        dict(name="sparse_decode", op="sparse", lanes=16, rows_lo=1, rows_hi=1, ctx_lo=8192, ctx_hi=131072, heads=32, kv=8, dim=128, page=64, top=64, dtype="bf16"),
        # verify blocks over a short and a long context, small pages
        dict(name="sparse_verify", op="sparse", lanes=5, rows_lo=2, rows_hi=5, ctx_lo=500, ctx_hi=40000, heads=12, kv=4, dim=64, page=32, top=40, dtype="f16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    heads, kv = rng.choice([(32, 8), (64, 8), (12, 4), (24, 4), (16, 16), (8, 1)])
    dim = rng.choice([64, 128, 128])
    page = rng.choice([16, 32, 64, 64, 128])
    base = dict(heads=heads, kv=kv, dim=dim, dtype=rng.choice(["bf16", "bf16", "f16"]))
    op = rng.choice(["norm_rope", "append", "attend", "attend", "attend", "sparse", "sparse"])
    if op == "norm_rope":
        return dict(op=op, tokens=_log(rng, 1, 8192), rot=rng.choice([dim, dim, dim // 2]), pairs=rng.random() < 0.3, **base)
    if op == "append":
        base.pop("heads")
        if rng.random() < 0.5:
            return dict(op=op, lanes=_log(rng, 1, 200), rows_lo=1, rows_hi=rng.randint(1, 6), ctx_lo=rng.randint(0, 60), ctx_hi=rng.randint(61, 500), page=page, **base)
        hi = _log(rng, 16, 1024)
        return dict(op=op, lanes=rng.randint(1, 12), rows_lo=rng.randint(1, 16), rows_hi=hi, ctx_lo=rng.randint(0, 9), ctx_hi=rng.randint(10, 1000), page=page, **base)
    if op == "attend":
        kind = rng.choice(["decode", "verify", "prefill"])
        if kind == "decode":
            lanes = _log(rng, 1, 64)
            hi = _log(rng, 64, min(1 << 20, (1 << 30) // (kv * dim * lanes)))
            return dict(op=op, lanes=lanes, rows_lo=1, rows_hi=1, ctx_lo=max(0, _log(rng, 1, hi) - 1), ctx_hi=hi, page=page, **base)
        if kind == "verify":
            lanes = _log(rng, 1, 32)
            hi = _log(rng, 64, min(1 << 19, (1 << 30) // (kv * dim * lanes)))
            return dict(op=op, lanes=lanes, rows_lo=rng.randint(1, 3), rows_hi=rng.randint(3, 9), ctx_lo=max(0, _log(rng, 1, hi) - 1), ctx_hi=hi, page=page, **base)
        hi = _log(rng, 32, 1024)
        return dict(op=op, lanes=rng.randint(1, 4), rows_lo=max(1, hi // rng.randint(1, 9)), rows_hi=hi, ctx_lo=0, ctx_hi=_log(rng, 8, 6000), page=page, **dict(base, heads=min(heads, 32)))
    lanes = _log(rng, 1, 16)
    hi = _log(rng, 600, min(131072, (1 << 31) // (kv * dim * lanes)))
    return dict(op=op, lanes=lanes, rows_lo=1, rows_hi=rng.choice([1, 1, 4, 6]), ctx_lo=_log(rng, 60, hi), ctx_hi=hi, page=page, top=rng.choice([8, 17, 32, 64]), **base)


def _spread(lo, hi, n):
    """n whole numbers from lo to hi, spread over their logarithm, in an order that is neither rising nor falling."""
    if n == 1:
        return [hi]
    a, b = math.log(lo + 1), math.log(hi + 1)
    v = [int(round(math.exp(a + (b - a) * i / (n - 1)))) - 1 for i in range(n)]
    step = next(s for s in (7, 5, 3, 11, 1) if math.gcd(s, n) == 1)
    return [v[(i * step) % n] for i in range(n)]


def _lens(case):
    rows = [max(1, r) for r in _spread(case["rows_lo"], case["rows_hi"], case["lanes"])]
    ctx = _spread(case["ctx_lo"], case["ctx_hi"], case["lanes"])[::-1]
    return rows, ctx


def work(case):
    d = case["dim"]
    g = case["kv"]
    if case["op"] == "norm_rope":
        n = case["tokens"] * (case["heads"] + g) * d
        return {"bytes": 4 * n + case["tokens"] * (4 * case["rot"] + 4), "flops": 8 * n}
    rows, ctx = _lens(case)
    page = case["page"]
    if case["op"] == "append":
        t = sum(rows)
        full = sum((c + r) // page - c // page for r, c in zip(rows, ctx))
        pages = sum((c + r - 1) // page - c // page + 1 for r, c in zip(rows, ctx))
        return {"bytes": t * g * d * 6 + 4 * t + full * g * (d + 4) + pages * g * 16, "flops": 4 * t * g * d}
    h = case["heads"]
    io = sum(rows) * h * (4 * d + 4)
    if case["op"] == "attend":
        kv = sum(r + c for r, c in zip(rows, ctx))
        pairs = sum(r * c + r * (r + 1) // 2 for r, c in zip(rows, ctx))
        return {"bytes": kv * g * d * 2 + sum(-(-(r + c) // page) for r, c in zip(rows, ctx)) * (8 * g + 4) + io, "flops": 4 * pairs * h * d}
    top = case["top"]
    blocks = [-(-(r + c) // page) for r, c in zip(rows, ctx)]
    read = sum(r * min(b, top) for r, b in zip(rows, blocks)) * page  # the rows of a block of a verify block may share what they read
    share = sum(min(b, top) for b in blocks) * page
    return {"bytes": share * g * d * 2 + sum(blocks) * g * (d + 4) + io + sum(rows) * g * top * 4,
            "flops": 4 * read * h * d + 2 * sum(r * b for r, b in zip(rows, blocks)) * g * d}


# ------------------------------------------------------------------------------------------------------------------
# Inputs
# ------------------------------------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(DEV).manual_seed(seed)


def _layout(case, gen):
    """cu_seqlens, positions, slots and block tables of the ragged batch; page 0 is the pool's scratch page."""
    rows, ctx = _lens(case)
    page, lanes = case["page"], case["lanes"]
    need = [-(-(r + c) // page) for r, c in zip(rows, ctx)]
    pages = 1 + sum(need)
    perm = 1 + torch.randperm(pages - 1, device=DEV, generator=gen)
    stride = max(need) + 1
    need_t = torch.tensor(need, device=DEV)
    first = torch.cumsum(need_t, 0) - need_t
    at = torch.arange(stride, device=DEV)
    bt = torch.where(at[None] < need_t[:, None], perm[(first[:, None] + at[None]).clamp(max=pages - 2)], 0)
    rows_t, ctx_t = torch.tensor(rows, device=DEV), torch.tensor(ctx, device=DEV)
    total = sum(rows)
    cu = torch.zeros(lanes + 1, dtype=torch.int64, device=DEV)
    cu[1:] = torch.cumsum(rows_t, 0)
    lane = torch.repeat_interleave(torch.arange(lanes, device=DEV), rows_t, output_size=total)
    row = torch.arange(total, device=DEV) - cu[lane]
    pos = ctx_t[lane] + row
    slots = bt[lane, pos // page] * page + pos % page
    i32 = dict(dtype=torch.int32)
    return dict(case=dict(case), pages=pages, lanes=lanes, total=total, max_rows=max(rows), max_kv=max(r + c for r, c in zip(rows, ctx)),
                bt=bt.to(**i32).contiguous(), cu=cu.to(**i32), pos=pos.to(**i32), slots=slots.to(**i32), lane=lane, row=row)


def _rope_table(rows, rot, base=10000.0):
    """cosines then sines of each position's angles, as hk_rope_table lays them out; angles in 64 bits."""
    f = base ** (-torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / rot)
    a = torch.arange(rows, device=DEV, dtype=torch.float64)[:, None] * f
    return torch.cat([a.cos(), a.sin()], 1).float().contiguous()


def _cache(case, s, gen):
    """A filled pool: e4m3 rows with a power-of-two scale for each page and head, as an append leaves them."""
    g, d, page = case["kv"], case["dim"], case["page"]
    shape = (s["pages"], g, page, d)
    for name, bias in (("k", 0.35), ("v", 0.0)):
        x = torch.randn(shape, device=DEV, generator=gen, dtype=torch.bfloat16)
        if bias:  # keys of neighbouring tokens are alike: a direction of each page's own
            x += torch.randn((s["pages"], g, 1, d), device=DEV, generator=gen, dtype=torch.bfloat16) * bias
        mag = torch.randint(6, 9, (s["pages"], g), device=DEV, generator=gen)  # 64 to 256 times the stored unit
        x *= torch.exp2(mag.float() - 1.5).to(torch.bfloat16)[:, :, None, None]
        s[name + "c"] = x.clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        s[name + "s"] = torch.exp2(-mag.float() + 1).contiguous()
        del x


def _centroids(kc, ks, page):
    """int8 centroid and its factor for every page and head: column sums of the stored values in units of 2^-9."""
    total = (kc.view(torch.float8_e4m3fn).to(torch.bfloat16).float() * 512).sum(2, dtype=torch.float64).float()
    top = total.abs().amax(-1)
    r = torch.where(top > 0, torch.full_like(top, 127) / top, torch.zeros_like(top))
    c = (total * r[..., None]).round().to(torch.int8)
    unit = torch.full_like(top, 127.0 * 512.0 * page)
    return c.contiguous(), (ks * (top / unit)).contiguous()


def prepare(case, seed):
    gen = _gen(seed)
    dt = DTYPES[case["dtype"]]
    g, d = case["kv"], case["dim"]

    def normal(*shape):
        return torch.randn(shape, device=DEV, generator=gen).to(dt)

    if case["op"] == "norm_rope":
        t, h = case["tokens"], case["heads"]
        x = normal(t, (h + 2 * g) * d)  # rows of a fused projection: queries, keys, values
        span = 16384
        return dict(case=dict(case), qkv=x, q=x[:, :h * d].view(t, h, d), k=x[:, h * d:(h + g) * d].view(t, g, d), qg=1 + 0.1 * normal(d), kg=1 + 0.1 * normal(d),
                    pos=torch.randint(0, span, (t,), device=DEV, generator=gen, dtype=torch.int32), table=_rope_table(span, case["rot"]))
    s = _layout(case, gen)
    _cache(case, s, gen)
    if case["op"] == "append":
        x = normal(s["total"], 2 * g * d)
        x[:, :g * d] *= 1.5
        s["k"], s["v"] = x[:, :g * d].view(-1, g, d), x[:, g * d:].view(-1, g, d)
        s["cen"] = torch.zeros((s["pages"], g, d), dtype=torch.int8, device=DEV)
        s["cs"] = torch.zeros((s["pages"], g), device=DEV)
        return s
    s["q"] = normal(s["total"], case["heads"], d) * 1.7
    s["scale"] = d ** -0.5
    if case["op"] == "sparse":
        s["cen"], s["cs"] = _centroids(s["kc"], s["ks"], case["page"])
    return s


# ------------------------------------------------------------------------------------------------------------------
# Plain forms
# ------------------------------------------------------------------------------------------------------------------

def _plain_norm_rope(x, gain, pos, table, rot, pairs, eps=1e-6):
    y = x.float()
    y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + eps) * gain.float()
    cs = table[pos.long()]
    c, n = cs[:, None, :rot // 2], cs[:, None, rot // 2:]
    if pairs:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
        r = torch.stack([a * c - b * n, b * c + a * n], -1).flatten(-2)
    else:
        a, b = y[..., :rot // 2], y[..., rot // 2:rot]
        r = torch.cat([a * c - b * n, b * c + a * n], -1)
    return torch.cat([r, y[..., rot:]], -1).to(x.dtype)


def _pow2_scale(top):
    """The least power of two s with top <= 448 s, for top >= 2^-32."""
    top = top.clamp(min=2.0 ** -32)
    m, e = torch.frexp(top)  # top = m 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    return torch.exp2((e - 9 + (m > 0.875).int()).double()).float()


def _f8(x):
    return x.to(torch.float8_e4m3fn)


def _plain_append(s):
    page, g = s["case"]["page"], s["case"]["kv"]
    slot = s["slots"].long()
    at, off = slot // page, slot % page
    lead = torch.ones_like(at, dtype=torch.bool)
    lead[1:] = at[1:] != at[:-1]
    run = torch.cumsum(lead, 0) - 1  # which run of rows in one page a row belongs to
    n = s["total"]  # at most so many runs; those past the last are all zeros and fall on the scratch page
    zero = torch.zeros(n, dtype=torch.int64, device=DEV)
    rpage = zero.index_put((run,), at)
    roff = torch.full((n,), page, device=DEV).scatter_reduce(0, run, off, "amin")
    rend = zero.scatter_reduce(0, run, off, "amax") + 1
    used = rpage > 0
    for x, cache, scale in ((s["k"], s["kc"], s["ks"]), (s["v"], s["vc"], s["vs"])):
        x = x.float()
        top = torch.zeros((n, g), device=DEV).scatter_reduce(0, run[:, None].expand(-1, g), x.abs().amax(-1), "amax")
        new = _pow2_scale(top)
        old = scale[rpage]
        kept = (roff > 0)[:, None]
        new = torch.where(kept, torch.maximum(old, new), new)
        rows = cache[rpage]  # (runs, kv, page, dim): the pages as they are, with the rows before the new ones brought to the new scale
        again = _f8(rows.view(torch.float8_e4m3fn).float() * (old / new)[..., None, None]).view(torch.uint8)
        before = (torch.arange(page, device=DEV)[None] < roff[:, None])[:, None, :, None] & (old < new)[..., None, None]
        rows = torch.where(before, again, rows)
        target = torch.where(used, rpage, 0)
        cache[target] = torch.where(used[:, None, None, None], rows, cache[0])
        scale[target] = torch.where(used[:, None], new, scale[0])
        q = _f8((x / scale[at][..., None]).clamp(-448, 448)).view(torch.uint8)
        cache[at, :, off] = q
    c, f = _centroids(s["kc"][rpage], s["ks"][rpage], page)
    full = used & (rend == page)
    target = torch.where(full, rpage, 0)
    s["cen"][target] = torch.where(full[:, None, None], c, s["cen"][0])
    s["cs"][target] = torch.where(full[:, None], f, s["cs"][0])
    return _append_outputs(s)


def _append_outputs(s):
    return dict(k=s["kc"].view(torch.float8_e4m3fn), v=s["vc"].view(torch.float8_e4m3fn), k_scale=s["ks"], v_scale=s["vs"], centroid=s["cen"], centroid_scale=s["cs"])


def _padded_rows(s):
    """The rows of each lane side by side: indices [lanes, max_rows], and which of them are rows."""
    cu = s["cu"].long()
    idx = cu[:-1, None] + torch.arange(s["max_rows"], device=DEV)
    return idx.clamp(max=s["total"] - 1), idx < cu[1:, None]


def _plain_blocks(s):
    case = s["case"]
    g, d, page, top = case["kv"], case["dim"], case["page"], case["top"]
    n = -(-s["max_kv"] // page)
    q = s["q"].double().view(s["total"], g, -1, d).sum(2).float()
    most = q.abs().amax(-1)
    r = torch.where(most > 0, torch.full_like(most, 127) / most, torch.zeros_like(most))
    qi = (q * r[..., None]).round()
    idx, _ = _padded_rows(s)
    pages = s["bt"][:, :n].long()
    dots = torch.einsum("lrgd,lngd->lrgn", qi[idx], s["cen"][pages].float())  # whole numbers below 2^22: exact in 32 bits
    score = (dots * s["cs"][pages].transpose(1, 2)[:, None])[s["lane"], s["row"]]
    last = (s["pos"].long() // page)[:, None, None]
    j = torch.arange(n, device=DEV)
    score = torch.where((j < SINK) | (j > last - LOCAL), math.inf, score)
    score = torch.where(j > last, -math.inf, score)
    val, order = torch.sort(score, dim=-1, descending=True, stable=True)
    ids = torch.where(val[..., :top] > -math.inf, order[..., :top], n)
    ids = torch.nn.functional.pad(ids, (0, max(0, top - n)), value=n).sort(-1)[0]
    return torch.where(ids < n, ids, -1).to(torch.int32)


def _plain_attend(s, blocks=None):
    case = s["case"]
    h, g, d, page = case["heads"], case["kv"], case["dim"], case["page"]
    grp, lanes, rows = h // g, s["lanes"], s["max_rows"]
    n = -(-s["max_kv"] // page)
    pages = s["bt"][:, :n].long()

    def values(c, f):
        x = c[pages].view(torch.float8_e4m3fn).float() * f[pages][..., None, None]
        return x.transpose(1, 2).reshape(lanes, g, n * page, d)

    idx, _ = _padded_rows(s)
    q = s["q"].float()[idx].view(lanes, rows, g, grp, d).transpose(1, 2).reshape(lanes, g, rows * grp, d)
    x = torch.matmul(q, values(s["kc"], s["ks"]).transpose(-1, -2)).view(lanes, g, rows, grp, n * page).mul_(s["scale"])
    seen = torch.arange(n * page, device=DEV) <= s["pos"].long()[idx][..., None]
    seen = seen[:, None, :, None]
    if blocks is not None:
        hit = torch.zeros((s["total"], g, n + 1), dtype=torch.bool, device=DEV)
        hit.scatter_(2, torch.where(blocks >= 0, blocks, n).long(), True)
        hit = hit[..., :n][idx].permute(0, 2, 1, 3).repeat_interleave(page, -1)
        seen = seen & hit[:, :, :, None]
    x.masked_fill_(~seen, -math.inf)
    m = x.amax(-1, keepdim=True)
    x = x.sub_(m).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(lanes, g, rows * grp, n * page), values(s["vc"], s["vs"])).view(lanes, g, rows, grp, d) / total
    lse = (m + total.log())[..., 0]
    o = o.permute(0, 2, 1, 3, 4).reshape(lanes, rows, h, d)[s["lane"], s["row"]]
    lse = lse.permute(0, 2, 1, 3).reshape(lanes, rows, h)[s["lane"], s["row"]]
    return o.to(s["q"].dtype), lse


# ------------------------------------------------------------------------------------------------------------------
# One pass
# ------------------------------------------------------------------------------------------------------------------

def _own(s):
    from hyperkernel_b200 import _lib as hk

    case = s["case"]
    if case["op"] == "norm_rope":
        return hk.qk_norm_rope(s["q"], s["k"], s["pos"], s["table"], s["qg"], s["kg"], interleaved=case["pairs"], eps=1e-6)
    if case["op"] == "append":
        hk.gqa_append_fp8(s["k"], s["v"], s["slots"], s["kc"], s["vc"], s["ks"], s["vs"], s["cen"], s["cs"])
        return _append_outputs(s)
    if case["op"] == "attend":
        return hk.gqa_decode_fp8(s["q"], s["kc"], s["vc"], s["ks"], s["vs"], s["bt"], s["cu"], s["pos"], s["max_rows"], s["max_kv"], s["scale"])
    blocks = hk.gqa_select_blocks(s["q"], s["cen"], s["cs"], s["bt"], s["cu"], s["pos"], case["page"], s["max_kv"], case["top"], sink=SINK, local=LOCAL)
    return (blocks, *hk.gqa_sparse_fp8(s["q"], s["kc"], s["vc"], s["ks"], s["vs"], s["bt"], s["cu"], s["pos"], blocks, s["scale"]))


def run(state):
    if own:
        return _own(state)
    case = state["case"]
    if case["op"] == "norm_rope":
        rest = (state["pos"], state["table"], case["rot"], case["pairs"])
        return _plain_norm_rope(state["q"], state["qg"], *rest), _plain_norm_rope(state["k"], state["kg"], *rest)
    if case["op"] == "append":
        return _plain_append(state)
    if case["op"] == "attend":
        return _plain_attend(state)
    blocks = _plain_blocks(state)
    return (blocks, *_plain_attend(state, blocks))


# ------------------------------------------------------------------------------------------------------------------
# The definitions in 64 bits, a lane and a head at a time
# ------------------------------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm_rope":
        return [_exact_norm_rope(x, gain, s, case) for x, gain in ((s["q"], s["qg"]), (s["k"], s["kg"]))]
    if case["op"] == "append":
        return _exact_append(s, case)
    return _exact_attend(s, case)


def _exact_norm_rope(x, gain, s, case):
    rot = case["rot"]
    x = x.double()
    y = x / ((x ** 2).sum(-1, keepdim=True) / x.shape[-1] + 1e-6).sqrt() * gain.double()
    z = torch.view_as_complex(s["table"][s["pos"].long()].double().view(-1, 2, rot // 2).transpose(1, 2).contiguous())[:, None]
    out = y.clone()
    i = torch.arange(rot // 2, device=DEV)
    a, b = (2 * i, 2 * i + 1) if case["pairs"] else (i, i + rot // 2)
    turned = torch.complex(y[..., a], y[..., b]) * z
    out[..., a], out[..., b] = turned.real, turned.imag
    return out


def _e4m3(x):
    """x rounded to e4m3, ties to even, saturating at 448; in 64 bits."""
    a = x.abs().clamp(max=448)
    step = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)
    return torch.sign(x) * (a / step).round() * step


def _exact_append(s, case):
    page, g = case["page"], case["kv"]
    kc, vc = (s[n].view(torch.float8_e4m3fn).double() for n in ("kc", "vc"))
    ks, vs = s["ks"].double(), s["vs"].double()
    cs = s["cs"].double()
    slots = s["slots"].tolist()
    t = 0
    while t < len(slots):
        p, o = divmod(slots[t], page)
        n = 1
        while t + n < len(slots) and slots[t + n] // page == p:
            n += 1
        for x, cache, scale in ((s["k"], kc, ks), (s["v"], vc, vs)):
            x = x[t:t + n].double().transpose(0, 1)
            top = x.abs().amax((1, 2)).clamp(min=2.0 ** -32)
            e = torch.ceil(torch.log2(top / 448))
            f = torch.exp2(e)
            f = torch.where(top > 448 * f, 2 * f, torch.where(top <= 224 * f, f / 2, f))
            if o > 0:
                f = torch.maximum(f, scale[p])
                cache[p, :, :o] = torch.where((f > scale[p])[:, None, None], _e4m3(cache[p, :, :o] * (scale[p] / f)[:, None, None]), cache[p, :, :o])
            scale[p] = f
            cache[p, :, o:o + n] = _e4m3(x / f[:, None, None])
        if o + n == page:
            cs[p] = ks[p] * (kc[p].sum(1).abs().amax(-1) / (127 * page))
        t += n
    return dict(k=kc, v=vc, k_scale=ks, v_scale=vs, centroid=None, centroid_scale=cs)


def _exact_blocks(s, case, t, pages):
    """The blocks of row t for every KV head: int8 dot products, rounded where the definition rounds to 32 bits."""
    g, d, top = case["kv"], case["dim"], case["top"]
    n = int(s["pos"][t]) // case["page"] + 1
    q = s["q"][t].double().view(g, -1, d).sum(1).float().double()
    most = q.abs().amax(-1)
    r = (127 / most.clamp(min=1e-300)).float().double() * (most > 0)
    qi = (q * r[:, None]).float().double().round()
    score = ((s["cen"][pages[:n]].double() * qi).sum(-1) * s["cs"][pages[:n]].double()).float()
    score[:SINK] = math.inf
    score[max(0, n - LOCAL):] = math.inf
    return [torch.sort(score[:, i], descending=True, stable=True)[1][:top].sort()[0] for i in range(g)]


def _exact_attend(s, case):
    h, g, d, page = case["heads"], case["kv"], case["dim"], case["page"]
    out = torch.zeros((s["total"], h, d), dtype=torch.float64, device=DEV)
    lse = torch.zeros((s["total"], h), dtype=torch.float64, device=DEV)
    cu = s["cu"].tolist()
    for b in range(s["lanes"]):
        t0, t1 = cu[b], cu[b + 1]
        pos = s["pos"][t0:t1].long()
        n = int(pos.max()) + 1
        pages = s["bt"][b, :-(-n // page)].long()
        sel = [_exact_blocks(s, case, t, pages) for t in range(t0, t1)] if case["op"] == "sparse" else None
        for i in range(g):
            k = (s["kc"][pages, i].view(torch.float8_e4m3fn).double() * s["ks"][pages, i].double()[:, None, None]).view(-1, d)[:n]
            v = (s["vc"][pages, i].view(torch.float8_e4m3fn).double() * s["vs"][pages, i].double()[:, None, None]).view(-1, d)[:n]
            hs = slice(i * (h // g), (i + 1) * (h // g))
            for a in range(t0, t1, 256):
                e = min(a + 256, t1)
                w = torch.einsum("thd,nd->thn", s["q"][a:e, hs].double(), k) * s["scale"]
                seen = torch.arange(n, device=DEV) <= pos[a - t0:e - t0, None]
                if sel is not None:
                    hit = torch.zeros((e - a, len(pages)), dtype=torch.bool, device=DEV)
                    for t in range(a, e):
                        hit[t - a, sel[t - t0][i]] = True
                    seen = seen & hit.repeat_interleave(page, 1)[:, :n]
                w = w.masked_fill(~seen[:, None], -math.inf)
                z = torch.logsumexp(w, -1)
                lse[a:e, hs] = z
                out[a:e, hs] = torch.einsum("thn,nd->thd", torch.exp(w - z[..., None]), v)
    return (None, out, lse) if case["op"] == "sparse" else (out, lse)
