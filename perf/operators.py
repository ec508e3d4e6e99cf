"""The full-attention operators of a serving step (``pla_b200.decode.full_attention``) as cases: block tables and slot
maps from request lengths, rotary positions, the per-head norm of queries and keys with the rotation and the cache
write, and the attention of one new token over the paged cache. ``own`` selects the library's calls; otherwise every
operator runs in its plain form, elementary torch operations in 32 bits (angles in 64)."""
import math

import torch

own = False

# (query heads, key/value heads): groups of 1 to 16, odd group sizes among them
HEADS = [(16, 2), (32, 8), (32, 4), (8, 8), (24, 8), (20, 4), (16, 1), (5, 1), (12, 2), (6, 3)]
# (head size, rotated part)
DIMS = [(64, 64), (96, 48), (128, 128), (128, 64), (192, 64), (256, 64), (256, 256), (128, 40)]
CACHE_CAP = 1.1e9          # bytes of keys and values that an attention case may read
ROWS_CAP = 32768 * 24 * 256   # elements of q, k and v that a rotation case may hold


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # a decode step's plan: 256 running requests (the batch of the repository's decode benchmark), a new page now and then
        dict(name="tables decode 256", op="tables", N=256, kind="decode", ctx=32768, new=1, block=64),
        # a prefill step's plan: eight packed sequences of 512 to 8,192 tokens (the prefill benchmark), nothing cached yet
        dict(name="tables prefill 8", op="tables", N=8, kind="prefill", ctx=0, new=8192, block=16),
        # the smallest decode step: one request's q and k, half layout, whole head
        dict(name="rotary 1 token", op="rotary", T=1, hq=32, hk=8, D=128, R=128, interleaved=False, dtype="bf16", far=4096),
        # a prefill chunk, interleaved, half of the head, positions far out in a long context
        dict(name="rotary 32761 interleaved", op="rotary", T=32761, hq=32, hk=8, D=128, R=64, interleaved=True, dtype="fp16", far=1048576),
        # a decode step of a hybrid layer: 256-wide heads, a quarter rotated, k and v into their pages
        dict(name="norm rotary cache decode 64", op="norm", cache=True, T=64, hq=16, hk=2, D=256, R=64, interleaved=False, dtype="bf16",
             far=131072, block=64, layout="separate", unit=True),
        # the same layer in a packed prefill of 32K tokens
        dict(name="norm rotary cache prefill 32K", op="norm", cache=True, T=32768, hq=16, hk=2, D=256, R=64, interleaved=False, dtype="bf16",
             far=32768, block=16, layout="packed", unit=True),
        # a mid-sized chunk whose k is kept dense (no cache), odd token count
        dict(name="norm rotary 1999", op="norm", cache=False, T=1999, hq=32, hk=8, D=128, R=128, interleaved=False, dtype="fp16", far=65536,
             block=16, layout="separate", unit=False),
        # one request with a short context: latency
        dict(name="attention 1 x 777", op="attention", B=1, hq=16, hk=2, D=128, longest=777, ragged=False, block=16, layout="separate", dtype="bf16"),
        # a small batch of ordinary contexts
        dict(name="attention 8 x 4K", op="attention", B=8, hq=32, hk=8, D=128, longest=4096, ragged=True, block=16, layout="packed", dtype="fp16"),
        # a full batch, ragged to 16K, 256-wide heads
        dict(name="attention 64 x 16K", op="attention", B=64, hq=16, hk=2, D=256, longest=16384, ragged=True, block=64, layout="separate", dtype="bf16"),
        # one very long context: all SMs on one request
        dict(name="attention 1 x 128K", op="attention", B=1, hq=32, hk=8, D=128, longest=131071, ragged=False, block=64, layout="separate", dtype="bf16"),
        # many short contexts, heads first in the page, small heads
        dict(name="attention 250 x 2K", op="attention", B=250, hq=32, hk=4, D=64, longest=2048, ragged=True, block=32, layout="heads", dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tables", "rotary", "norm", "norm", "attention", "attention", "attention"])
    dtype = rng.choice(["bf16", "fp16"])
    block = rng.choice([1, 8, 16, 32, 48, 64, 128, 256])
    layout = rng.choice(["separate", "packed", "heads"])
    if op == "tables":
        kind = rng.choice(["decode", "prefill", "mixed"])
        N = _log(rng, 1, 1024 if kind == "decode" else 64)
        new = 1 if kind == "decode" else _log(rng, 1, max(1, min(8192, 65536 // N)))
        return dict(op=op, N=N, kind=kind, ctx=0 if kind == "prefill" else _log(rng, 1, 65536), new=new, block=max(block, 8))
    hq, hk = rng.choice(HEADS)
    if op == "attention":
        D = rng.choice([64, 96, 128, 192, 256])
        B = _log(rng, 1, 256)
        most = int(CACHE_CAP / (B * hk * D * 4))
        return dict(op=op, B=B, hq=hq, hk=hk, D=D, longest=min(_log(rng, 1, 131072), most), ragged=rng.random() < 0.7, block=block, layout=layout, dtype=dtype)
    D, R = rng.choice(DIMS)
    T = min(_log(rng, 1, 32768), ROWS_CAP // ((hq + 2 * hk) * D))
    far = _log(rng, 1024, 1 << 20)
    inter = rng.random() < 0.4
    if op == "rotary":
        return dict(op=op, T=T, hq=hq, hk=hk, D=D, R=R, interleaved=inter, dtype=dtype, far=far)
    return dict(op=op, cache=rng.random() < 0.7, T=T, hq=hq, hk=hk, D=D, R=R, interleaved=inter, dtype=dtype, far=far, block=block,
                layout=layout, unit=rng.random() < 0.5)


# ------------------------------------------------------------------------------------------------ lengths of a case
def _spread(n, lo, hi):
    """n lengths between lo and hi, evenly spread and mixed, the first one hi: the same for every seed, so that the work is."""
    return [hi - int((hi - lo) * ((i * 0.6180339887498949) % 1.0)) for i in range(n)]


def _table_lengths(c):
    N, new, ctx = c["N"], c["new"], c["ctx"]
    if c["kind"] == "prefill":
        return [0] * N, _spread(N, max(1, new // 16), new)
    if c["kind"] == "decode":
        return _spread(N, max(1, ctx // 8), ctx), [1] * N
    old = _spread(N, 0, ctx)
    return [0 if i % 3 == 1 else old[i] for i in range(N)], [n if i % 2 else 1 for i, n in enumerate(_spread(N, 1, new))]


def _attention_lengths(c):
    """Ragged batches end in a row of length zero, as a padded captured batch has it."""
    if not c["ragged"]:
        return [c["longest"]] * c["B"]
    out = _spread(c["B"], max(1, c["longest"] // 16), c["longest"])
    if c["B"] > 4:
        out[-1] = 0
    return out


# ------------------------------------------------------------------------------------------------ inputs
def _dtype(c):
    return torch.bfloat16 if c["dtype"] == "bf16" else torch.float16


def _cache(blocks, c, g):
    """Keys and values in pages: two tensors, two halves of one, or pages with the heads first; always addressed [page, token, head, :]."""
    bs, hk, D = c["block"], c["hk"], c["D"]
    kw = dict(device="cuda", dtype=_dtype(c), generator=g)
    if c["layout"] == "packed":
        both = torch.randn(blocks, 2, bs, hk, D, **kw)
        return both[:, 0], both[:, 1]
    if c["layout"] == "heads":
        return torch.randn(blocks, hk, bs, D, **kw).transpose(1, 2), torch.randn(blocks, hk, bs, D, **kw).transpose(1, 2)
    return torch.randn(blocks, bs, hk, D, **kw), torch.randn(blocks, bs, hk, D, **kw)


def _table(pages, columns, g, spare=3):
    """A block table whose rows hold `pages[n]` pages of a shuffled pool, -1 behind them; and the pool's size."""
    pages = torch.tensor(pages, device="cuda")
    blocks = int(pages.sum()) + spare
    order = torch.randperm(blocks, device="cuda", generator=g).to(torch.int32)
    col = torch.arange(columns, device="cuda")
    at = (pages.cumsum(0) - pages)[:, None] + col
    table = torch.where(col < pages[:, None], order[at.clamp(max=blocks - 1)], -1)
    return table.to(torch.int32), order, blocks


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    i32 = dict(device="cuda", dtype=torch.int32)
    if c["op"] == "tables":
        ctx, new = _table_lengths(c)
        turn = int(torch.randperm(len(ctx), device="cuda", generator=g)[0])
        ctx, new = ctx[turn:] + ctx[:turn], new[turn:] + new[:turn]
        bs = c["block"]
        held = [-(-x // bs) for x in ctx]
        columns = max(-(-(x + y) // bs) for x, y in zip(ctx, new)) + 2
        wanted = sum(-(-(x + y) // bs) - h for x, y, h in zip(ctx, new, held))
        table, order, blocks = _table(held, columns, g, spare=wanted + 7)
        free = order[sum(held):].contiguous()
        qsl = torch.tensor([0] + new, **i32).cumsum(0).to(torch.int32)
        return dict(c=c, table=table, ctx=torch.tensor(ctx, **i32), qsl=qsl, free=free, tokens=sum(new),
                    start=torch.tensor([2], **i32))
    dt = _dtype(c)
    if c["op"] == "attention":
        lens = _attention_lengths(c)
        turn = int(torch.randperm(len(lens), device="cuda", generator=g)[0])
        lens = lens[turn:] + lens[:turn]
        columns = -(-c["longest"] // c["block"])
        table, _, blocks = _table([-(-n // c["block"]) for n in lens], columns, g)
        k, v = _cache(blocks, c, g)
        q = torch.randn(c["B"], c["hq"], c["D"], device="cuda", dtype=dt, generator=g) * 1.5
        return dict(c=c, q=q, k=k, v=v, table=table, lens=torch.tensor(lens, **i32), scale=c["D"] ** -0.5)
    T, hq, hk, D, R = c["T"], c["hq"], c["hk"], c["D"], c["R"]
    row = torch.randn(T, (hq + 2 * hk) * D, device="cuda", dtype=dt, generator=g)   # a packed projection's row
    q, k, v = (x.unflatten(1, (-1, D)) for x in row.split([hq * D, hk * D, hk * D], dim=1))
    turns = 10000.0 ** (-torch.arange(0, R, 2, device="cuda", dtype=torch.float64) / R)
    s = dict(c=c, q=q, k=k, v=v, freq=turns, pos=torch.randint(0, c["far"], (T,), device="cuda", generator=g))
    if c["op"] == "norm":
        for w in ("qw", "kw"):
            s[w] = (torch.randn(D, device="cuda", generator=g) * 0.1 + (0.0 if c["unit"] else 1.0)).to(dt)
        if c["cache"]:
            blocks = -(-T // c["block"]) + 3
            s["kc"], s["vc"] = _cache(blocks, c, g)
            s["slots"] = torch.randperm(blocks * c["block"], device="cuda", generator=g)[:T]
            s["slots"][T // 2] = -1 if T > 4 else s["slots"][T // 2]           # a padding row
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_tables(s):
    table, ctx, qsl, free, bs = s["table"], s["ctx"].long(), s["qsl"].long(), s["free"], s["c"]["block"]
    N, C = table.shape
    new = qsl[1:] - qsl[:-1]
    held = (ctx + bs - 1) // bs
    need = ((ctx + new + bs - 1) // bs).clamp(max=C) - held
    base = s["start"].long() + need.cumsum(0) - need
    col = torch.arange(C, device=table.device) - held[:, None]
    at = base[:, None] + col
    page = torch.where(at < free.numel(), free[at.clamp(0, free.numel() - 1)], -1)
    table.copy_(torch.where((col >= 0) & (col < need[:, None]), page, table))
    t = torch.arange(s["tokens"], device=table.device)
    n = torch.searchsorted(qsl[1:], t, right=True).clamp(max=N - 1)
    pos = ctx[n] + t - qsl[n]
    page = table[n, (pos // bs).clamp(max=C - 1)].long()
    slots = torch.where((page >= 0) & (pos // bs < C), page * bs + pos % bs, -1)
    return dict(table=table, slots=slots, positions=pos, seq_lens=(ctx + new).to(torch.int32),
                free_next=(s["start"] + need.sum()).clamp(max=free.numel()).to(torch.int32))


def _rotate(x, cos, sin, R, interleaved):
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., :R // 2], x[..., R // 2:R])
    u, v = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([u, v], -1).flatten(-2) if interleaved else torch.cat([u, v], -1)
    return torch.cat([turned, x[..., R:]], -1)


def _plain_rotary(s, weights):
    c, dt = s["c"], s["q"].dtype
    angle = s["pos"].double()[:, None] * s["freq"]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    out = []
    for x, w in ((s["q"], "qw"), (s["k"], "kw")):
        x = x.float()
        if weights:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * (s[w].float() + (1.0 if c["unit"] else 0.0))
        out.append(_rotate(x, cos, sin, c["R"], c["interleaved"]).to(dt))
    return out


def _plain_attention(s):
    q, k, v, table, lens, bs = s["q"], s["k"], s["v"], s["table"].long().clamp(min=0), s["lens"].long(), s["c"]["block"]
    B, hq, D = q.shape
    hk = k.size(2)
    L = s["c"]["longest"]
    t = torch.arange(L, device=q.device)
    page, off = table[:, t // bs], (t % bs).expand(B, L)
    live = t < lens[:, None]
    score = torch.einsum("bhgd,blhd->bhgl", q.float().view(B, hk, hq // hk, D), k[page, off].float()) * s["scale"]
    score = score.masked_fill(~live[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    out = torch.einsum("bhgl,blhd->bhgd", p, v[page, off].float()) / total.clamp(min=1e-30)
    lse = (top + torch.log(total)).masked_fill(total == 0, -math.inf)
    return dict(out=out.reshape(B, hq, D).to(q.dtype), lse=lse.view(B, hq))


def _plain(s):
    op = s["c"]["op"]
    if op == "tables":
        return _plain_tables(s)
    if op == "attention":
        return _plain_attention(s)
    q, k = _plain_rotary(s, op == "norm")
    if op == "norm" and s["c"]["cache"]:
        slots, bs = s["slots"], s["c"]["block"]
        live = (slots >= 0).nonzero()[:, 0]
        s["kc"][slots[live] // bs, slots[live] % bs] = k[live]
        s["vc"][slots[live] // bs, slots[live] % bs] = s["v"][live]
        return dict(q=q, k_cache=s["kc"], v_cache=s["vc"])
    return dict(q=q, k=k)


# ------------------------------------------------------------------------------------------------ the library's calls
def _library(s):
    from pla_b200.decode import full_attention as fa
    c = s["c"]
    if c["op"] == "tables":
        p = fa.build_block_tables(s["table"], s["ctx"], s["qsl"], s["free"], c["block"], num_tokens=s["tokens"], free_start=s["start"])
        return dict(table=p.block_table, slots=p.slot_mapping, positions=p.positions, seq_lens=p.seq_lens, free_next=p.free_next)
    if c["op"] == "attention":
        out, lse = fa.paged_attention_decode(s["q"], s["k"], s["v"], s["table"], s["lens"], scale=s["scale"], return_lse=True)
        return dict(out=out, lse=lse)
    if c["op"] == "rotary":
        q, k = fa.apply_rotary(s["q"], s["k"], s["pos"], s["freq"], interleaved=c["interleaved"])
        return dict(q=q, k=k)
    if c["cache"]:
        q = fa.qk_norm_rotary_cache(s["q"], s["k"], s["v"], s["qw"], s["kw"], s["pos"], s["freq"], s["kc"], s["vc"], s["slots"],
                                    interleaved=c["interleaved"], unit_offset=c["unit"])
        return dict(q=q, k_cache=s["kc"], v_cache=s["vc"])
    q, k = fa.qk_norm_rotary(s["q"], s["k"], s["qw"], s["kw"], s["pos"], s["freq"], interleaved=c["interleaved"], unit_offset=c["unit"])
    return dict(q=q, k=k)


def run(state):
    return _library(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    if c["op"] == "tables":
        ctx, new = _table_lengths(c)
        bs = c["block"]
        pages = sum(-(-(x + y) // bs) - (-(-x // bs)) for x, y in zip(ctx, new))
        # lengths and offsets in, taken pages in and out, one held page per request that fills it up, slots, positions and lengths out
        return dict(bytes=4 * (2 * c["N"] + 1) + 8 * pages + 4 * sum(x % bs > 0 for x in ctx) + 16 * sum(new) + 4 * c["N"] + 8, flops=0)
    if c["op"] == "attention":
        total, D = sum(_attention_lengths(c)), c["D"]
        pages = sum(-(-n // c["block"]) for n in _attention_lengths(c))
        rows = c["B"] * c["hq"]
        return dict(bytes=4 * total * c["hk"] * D + 4 * rows * D + 4 * rows + 4 * pages + 4 * c["B"], flops=4 * total * c["hq"] * D)
    T, hq, hk, D, R = c["T"], c["hq"], c["hk"], c["D"], c["R"]
    rows = hq + hk
    size = 4 * T * rows * D + 8 * T + 4 * R
    flops = 3 * T * rows * R
    if c["op"] == "norm":
        size += 4 * D
        flops += 4 * T * rows * D
        if c["cache"]:
            size += 4 * T * hk * D + 8 * T
    return dict(bytes=size, flops=flops)


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    c = s["c"]
    if c["op"] == "tables":
        return None                                                     # whole numbers: they have to be equal
    if c["op"] == "attention":
        q, lens, bs = s["q"].double(), s["lens"].tolist(), c["block"]
        out, lse = torch.zeros_like(q), torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
        group = c["hq"] // c["hk"]
        for b, n in enumerate(lens):
            if n == 0:
                continue
            pages = s["table"][b, :-(-n // bs)].long()
            keys, values = (x[pages].flatten(0, 1)[:n].double() for x in (s["k"], s["v"]))
            for h in range(c["hk"]):
                z = (q[b, h * group:(h + 1) * group] @ keys[:, h].T) * s["scale"]
                lse[b, h * group:(h + 1) * group] = torch.logsumexp(z, -1)
                out[b, h * group:(h + 1) * group] = torch.softmax(z, -1) @ values[:, h]
        return dict(out=out, lse=lse)
    R = c["R"]
    wave = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s["pos"].double()[:, None] * s["freq"])[:, None]
    res = {}
    for key, w in (("q", "qw"), ("k", "kw")):
        x = s[key].double()
        if c["op"] == "norm":
            x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / c["D"] + 1e-6)
            x = x * (s[w].double() + 1.0 if c["unit"] else s[w].double())
        y = x.clone()
        first, second = (slice(0, R, 2), slice(1, R, 2)) if c["interleaved"] else (slice(0, R // 2), slice(R // 2, R))
        z = torch.complex(x[..., first], x[..., second]) * wave
        y[..., first], y[..., second] = z.real, z.imag
        res[key] = y
    if c["op"] == "norm" and c["cache"]:
        kc, vc, k = s["kc"].double(), s["vc"].double(), res["k"]
        to = s["slots"].tolist()
        rows = torch.tensor([t for t, x in enumerate(to) if x >= 0], device="cuda")
        page = torch.tensor([x // c["block"] for x in to if x >= 0], device="cuda")
        off = torch.tensor([x % c["block"] for x in to if x >= 0], device="cuda")
        kc[page, off], vc[page, off] = k[rows], s["v"][rows].double()
        return dict(q=res["q"], k_cache=kc, v_cache=vc)
    return res
