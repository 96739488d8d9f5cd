"""Cases for serving many long sequences from the paged 8-bit KV cache.

Four operators: attention of a batch whose sequences share a long prefix in
groups ("shared"), the attention weight that every cached row has received,
added up ("weigh"), eviction of the rows with the least of it ("evict"), and
rotary positions with several axes, given for every token because the row of
an evicted cache no longer says where a token stood ("rotate").

The cache (one layer): codes int8 ``[pages, Hkv, page, D]``, scales float32
``[pages, Hkv]`` for K and for V, and a table int32 ``[B, max_pages]`` with
the pool page of every ``page`` consecutive rows of a sequence.
"""
import math
import random

import torch

own = False

ROPE_BASE = 1e7     # of the decode stack


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # four answers sampled from one prompt, early in the answer
        dict(name="shared_samples", op="shared", batch=4, groups=1, L=1, kv_heads=2, rep=8,
             dim=256, page=64, prefix=2048, tail=173, ragged=False),
        # a server's decode step: three system prompts, answers of mixed lengths, idle slots
        dict(name="shared_prompts", op="shared", batch=48, groups=3, L=1, kv_heads=8, rep=4,
             dim=128, page=32, prefix=6400, tail=1501, ragged=True),
        # a verify step of 64 sequences behind one long document
        dict(name="shared_document", op="shared", batch=64, groups=1, L=4, kv_heads=2, rep=8,
             dim=256, page=64, prefix=32768, tail=1030, ragged=True),
        # a decode step of one sequence through the decode stack's attention layer
        dict(name="weigh_one", op="weigh", batch=1, L=1, kv_heads=2, rep=8, dim=256, page=64,
             keys=901, ragged=False),
        # a decode step of a batch of sequences of mixed lengths, some slots idle
        dict(name="weigh_batch", op="weigh", batch=32, L=1, kv_heads=8, rep=4, dim=128, page=32,
             keys=8190, ragged=True),
        # the last 64 rows of a long prompt weigh all of its rows
        dict(name="weigh_window", op="weigh", batch=1, L=64, kv_heads=2, rep=8, dim=256, page=64,
             keys=32768, ragged=False),
        # a sequence that has outgrown its 4096 rows by 64
        dict(name="evict_one", op="evict", batch=1, kv_heads=2, dim=256, page=64, rows=4160,
             keep=4096, first=64, recent=256, ragged=False, again=True),
        # a batch of them, each over its share by its own number of rows
        dict(name="evict_batch", op="evict", batch=32, kv_heads=8, dim=128, page=32, rows=2111,
             keep=2048, first=4, recent=128, ragged=True, again=True),
        # long prompts, written whole, down to what decoding keeps of them
        dict(name="evict_prompt", op="evict", batch=2, kv_heads=2, dim=256, page=64, rows=65536,
             keep=8192, first=64, recent=1024, ragged=False, again=False),
        # the rows of one verify step
        dict(name="rotate_step", op="rotate", batch=1, L=4, heads=16, kv_heads=2, dim=256, rope=64,
             sections="12,10,10", woven=False, norm=True, far=90000),
        # a prompt of text and images, heads rotated over all of their dims
        dict(name="rotate_images", op="rotate", batch=2, L=8191, heads=32, kv_heads=8, dim=128,
             rope=128, sections="24,20,20", woven=True, norm=False, far=5000),
        # a long prompt through the decode stack's attention layer
        dict(name="rotate_prompt", op="rotate", batch=1, L=65536, heads=16, kv_heads=2, dim=256,
             rope=64, sections="12,10,10", woven=False, norm=True, far=1000000),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("shared", "shared", "weigh", "evict", "rotate"))
    if op == "rotate":
        dim = rng.choice((64, 80, 96, 128, 192, 256))
        rope = rng.choice([r for r in (32, 64, 80, 96, 128, 256) if r <= dim])
        n = rng.choice((1, 2, 3, 3, 4))
        cuts = sorted(rng.randint(0, rope // 2) for _ in range(n - 1))
        sections = [b - a for a, b in zip([0] + cuts, cuts + [rope // 2])]
        heads = rng.choice((1, 2, 4, 8))
        case = dict(op=op, heads=heads * rng.choice((1, 2, 4, 7, 8)), kv_heads=heads, dim=dim,
                    rope=rope, sections=",".join(map(str, sections)), woven=rng.random() < 0.5,
                    norm=rng.random() < 0.5, far=_log_int(rng, 10, 10000000))
        case["batch"] = _log_int(rng, 1, 32)
        most = 65536 * 18 * 256 // ((case["heads"] + heads) * dim * case["batch"])
        case["L"] = _log_int(rng, 1, min(65536, most))
        return case
    base = dict(op=op, kv_heads=rng.choice((1, 2, 4, 8)), dim=rng.choice((64, 128, 256)),
                page=rng.choice((16, 32, 64, 128)), ragged=rng.random() < 0.6)
    width = base["kv_heads"] * base["dim"]
    if op == "evict":
        base["batch"] = _log_int(rng, 1, 32)
        most = 131072 * 512 // (width * base["batch"])
        again = rng.random() < 0.6
        rows = _log_int(rng, 40, max(64, min(65536, most // (4 if again else 1))))
        keep = rows - _log_int(rng, 1, max(1, min(256, rows // 4))) if again else \
            _log_int(rng, 20, max(21, rows // 2))
        first = rng.choice((0, 1, 4, keep // 8))
        base.update(rows=rows, keep=keep, first=first, recent=rng.choice((0, 1, keep // 8, keep // 2)),
                    again=again)
        return base
    base.update(rep=rng.choice((1, 2, 3, 4, 5, 7, 8, 16)))
    if op == "weigh":
        base["batch"] = _log_int(rng, 1, 32)
        L = rng.choice((1, 1, 1, 2, 4, 5, 8, 16, 33, 64))
        if L > 8:
            base["batch"] = min(base["batch"], 4)
        pairs = 32768 * 64 * 16 * 256 // (L * base["rep"] * width * base["batch"])
        most = max(64, L, min(131072 * 512 // (width * base["batch"]), 131072, pairs))
        base.update(L=L, keys=_log_int(rng, max(16, L), most))
        return base
    batch = _log_int(rng, 2, 64)
    base.update(batch=batch, groups=rng.choice((1, 1, 1, 2, 3, 5)), L=rng.choice((1, 1, 1, 2, 4, 5)))
    base["groups"] = min(base["groups"], batch // 2)
    pairs = 32768 * 64 * 64 * 256 // (base["L"] * base["rep"] * width * batch)
    most = max(2 * base["page"], min(32768, pairs, 64 * 32768 * 512 // (width * batch)))
    base["prefix"] = _log_int(rng, base["page"], most) // base["page"] * base["page"]
    base["tail"] = _log_int(rng, base["L"], max(64, min(1500, 64 * 1030 * 512 // (width * batch))))
    return base


# ------------------------------------------------------------ sizes of a case
def _groups(case):
    """(first sequence, sequences, rows of the prefix) of every group, from the case alone."""
    B, G, page = case["batch"], case["groups"], case["page"]
    if G == 1:
        return [(0, B, case["prefix"])]
    r = random.Random(7 * B + G)
    alone = 1 if case["ragged"] and B > 2 * G else 0   # the last sequence shares nothing
    ends = [(B - alone) * (g + 1) // G for g in range(G)]
    got, at = [], 0
    for g, end in enumerate(ends):
        pages = case["prefix"] // page
        got.append((at, end - at, page * (pages if g == 0 else max(1, int(pages * r.random())))))
        at = end
    return got


def _prefixes(case):
    of = [0] * case["batch"]
    for first, count, rows in _groups(case):
        of[first:first + count] = [rows] * count
    return of


def _lengths(case):
    """Per sequence (query rows of this pass, keys with them), from the case alone."""
    B = case["batch"]
    if case["op"] == "evict":
        r = random.Random(3 * case["rows"] + B)
        got = []
        for b in range(B):
            if not case["ragged"] or b == 0:
                got.append(case["rows"])
            elif b % 8 == 5:  # still within its share
                got.append(r.randint(0, case["keep"]))
            else:
                got.append(r.randint(case["keep"], case["rows"]))
        return [(0, n) for n in got]
    L = case["L"]
    if case["op"] == "shared":
        before, start = max(0, case["tail"] - L), _prefixes(case)
    else:
        before, start = max(0, case["keys"] - L), [0] * B
    r = random.Random(1000003 * L + 101 * before + B)
    got = []
    for b in range(B):
        if not case["ragged"] or b == 0:
            got.append((L, start[b] + before + L))
        elif b % 8 == 5:
            got.append((0, 0))  # an idle slot of the batch
        else:
            n = r.randint(max(1, L // 4), L)
            got.append((n, start[b] + n + int(before * r.uniform(0.02, 1.0))))
    return got


def _visible(case):
    """(query, key) pairs of one query head over the batch."""
    return sum(n * (keys - n) + n * (n + 1) // 2 for n, keys in _lengths(case))


def work(case):
    if case["op"] == "rotate":
        n = case["batch"] * case["L"] * (case["heads"] + case["kv_heads"])
        axes = len(case["sections"].split(","))
        return {"bytes": 4 * n * case["dim"] + 4 * axes * case["batch"] * case["L"],
                "flops": n * (3 * case["rope"] + (4 * case["dim"] if case["norm"] else 0))}
    width = case["kv_heads"] * case["dim"]
    lens = _lengths(case)
    if case["op"] == "evict":
        moved, scanned, held = 0.0, 0, 0
        for _, n in lens:
            held += min(n, case["keep"])
            over = n - case["keep"]
            if over > 0:
                scanned += n
                late = min(case["recent"], over)
                free = n - case["first"] - case["recent"]
                share = (case["keep"] - case["first"] - case["recent"]) / free if free > 0 else 1.0
                moved += late + (over - late) * max(0.0, share)
        # weights and positions looked at, rows moved (K and V, in and out), and the rows that
        # are held read back (codes in, bf16 out, zeros behind short sequences)
        return {"bytes": int(case["kv_heads"] * (8 * scanned + 16 * moved) + 4 * width * moved
                             + 2 * width * (held + 2 * case["batch"] * case["keep"])),
                "flops": int(2 * width * (moved + held))}
    heads = case["kv_heads"] * case["rep"]
    if case["op"] == "weigh":
        keys = sum(k for n, k in lens if n)
        new = sum(n for n, _ in lens)
        return {"bytes": width * keys + case["kv_heads"] * (8 * keys + 4 * new)
                + new * heads * (2 * case["dim"] + 4),
                "flops": 2 * case["dim"] * heads * _visible(case)}
    start = _prefixes(case)
    keys = sum(k - start[b] for b, (n, k) in enumerate(lens) if n)
    keys += sum(rows for first, count, rows in _groups(case)
                if any(n for n, _ in lens[first:first + count]))
    io = case["batch"] * heads * case["L"] * (4 * case["dim"] + 4)
    return {"bytes": 2 * width * keys + io, "flops": 4 * case["dim"] * heads * _visible(case)}


# ------------------------------------------------------------------- inputs
def _cache(case, g, lens, device):
    """A cache with room for every sequence, its pages in shuffled order; the sequences of a
    group have the pages of their prefix in common."""
    page, H, D, B = case["page"], case["kv_heads"], case["dim"], case["batch"]
    width = max(k for _, k in lens) // page + 1
    pages = B * width + 1  # the last page is in no table
    table = torch.randperm(B * width, generator=g, device=device).view(B, width).to(torch.int32)
    for first, count, rows in _groups(case) if case["op"] == "shared" else ():
        table[first:first + count, :rows // page] = table[first, :rows // page].clone()
    shape = (pages, H, page, D)
    c = {"table": table, "page": page}
    for name in ("k", "v"):
        codes = torch.empty(shape, dtype=torch.int8, device=device)
        step = max(1, (1 << 26) // (H * page * D))
        for i in range(0, pages, step):  # normal values, as the quantiser leaves them
            part = codes[i:i + step]
            part.copy_((torch.randn(part.shape, generator=g, device=device) * 36.0)
                       .round_().clamp_(-127, 127))
        c[name + "_codes"] = codes
        # amplitudes of pages differ by a factor of about two
        c[name + "_scales"] = (torch.rand((pages, H), generator=g, device=device) + 0.5) / 32.0
    return c


def _positions(case, g, device):
    """[axes, B, L]: text (all axes alike) with images in it, whose patches share a time and
    are counted along height and width."""
    A, B, L = len(case["sections"].split(",")), case["batch"], case["L"]
    start = torch.randint(0, case["far"], (B, 1), generator=g, device=device)
    i = torch.arange(L, device=device)[None]
    side = 24
    image, patch = i // 1024 * 1024, i % 1024 - (1024 - side * side)
    inside = (patch >= 0).expand(B, L)
    got = []
    for a in range(A):
        at = 0 * patch if a == 0 else patch // side if a == 1 else patch % side
        got.append(start + torch.where(inside, image + at, i))
    return torch.stack(got).to(torch.int32)


def _pair_axes(case):
    """The axis of every rotated pair: section after section, or dealt out in turn."""
    left = [int(n) for n in case["sections"].split(",")]
    if not case["woven"]:
        return tuple(a for a, n in enumerate(left) for _ in range(n))
    return tuple(a for k in range(max(left)) for a, n in enumerate(left) if k < n)


def prepare(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    s = dict(case=case)
    if case["op"] == "rotate":
        B, L, D = case["batch"], case["L"], case["dim"]
        # rows as a projection leaves them: the heads of a token side by side
        for name, heads in (("q", case["heads"]), ("k", case["kv_heads"])):
            x = torch.randn((B, L, heads, D), generator=g, device=device).to(torch.bfloat16)
            s[name] = x.transpose(1, 2)
            w = 1.0 + 0.1 * torch.randn(D, generator=g, device=device)
            s[name + "_norm"] = w.to(torch.bfloat16) if case["norm"] else None
        s["positions"] = _positions(case, g, device)
        s["axes"] = _pair_axes(case)
        if own:
            import vates_b200.rotary  # noqa: F401
        return s
    lens = _lengths(case)
    s["cache"] = _cache(case, g, lens, device)
    B, H, D = case["batch"], case["kv_heads"], case["dim"]
    s["rows"] = torch.tensor([n for n, _ in lens], dtype=torch.int32, device=device)
    s["lens"] = torch.tensor([k for _, k in lens], dtype=torch.int32, device=device)
    s["starts"] = _prefixes(case) if case["op"] == "shared" else None
    if case["op"] != "shared":
        room = s["cache"]["table"].shape[1] * case["page"]
        # what rows have received so far: a few have most of it
        s["weights"] = torch.randn((B, H, room), generator=g, device=device).mul_(2.0).exp_()
        if case["op"] == "evict" and case["again"]:
            # evicted from before: older rows in any order, the newest behind them
            old = torch.rand((B, H, case["keep"]), generator=g, device=device).argsort(-1)
            new = torch.arange(case["keep"], room, device=device).expand(B, H, -1)
            s["positions"] = torch.cat((old, new), -1).to(torch.int32)
        else:
            s["positions"] = torch.arange(room, device=device, dtype=torch.int32).expand(
                B, H, room).contiguous()
    if case["op"] != "evict":
        q = torch.randn((B, H * case["rep"], case["L"], D), generator=g, device=device)
        s["q"] = (q * 1.5).to(torch.bfloat16)
    if case["op"] == "weigh":
        s["seen"] = s["lens"] + 1000  # tokens of the sequence, with those evicted earlier
        s["lse"] = _lse(s)
    if own:
        from vates_b200.kv8 import PagedKV8Cache, SharedPrefix
        c = s["cache"]
        s["handle"] = PagedKV8Cache(c["k_codes"], c["v_codes"], c["k_scales"], c["v_scales"],
                                    c["table"])
        if case["op"] == "shared":
            s["plan"] = SharedPrefix(s["handle"], _groups(case))
    return s


# ---------------------------------------------------------------- plain form
def _rows(c, name, n):
    """float32 [B, H, n (whole pages), D]."""
    ids = c["table"][:, :-(-n // c["page"])].long()
    x = c[name + "_codes"][ids].float() * c[name + "_scales"][ids][..., None, None]
    B, P, H, page, D = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(B, H, P * page, D)


def _scores(s):
    """Masked scores [B, H, rep, L, keys] in float32."""
    case, c = s["case"], s["cache"]
    B, Hq, L, D = s["q"].shape
    H, rep = case["kv_heads"], case["rep"]
    k = _rows(c, "k", c["table"].shape[1] * c["page"])
    S = k.shape[2]
    z = (s["q"].float().view(B, H, rep * L, D) @ k.transpose(-1, -2)).mul_(D ** -0.5)
    z = z.view(B, H, rep, L, S)
    i = torch.arange(L, device=z.device)
    last = (s["lens"] - s["rows"])[:, None] + i + 1
    last = torch.where(i < s["rows"][:, None], last, 0)                       # keys seen by row i
    hidden = torch.arange(S, device=z.device) >= last[..., None]              # [B, L, S]
    return z.masked_fill_(hidden[:, None, None], -math.inf)


def _normaliser(z):
    top = z.amax(-1, keepdim=True)
    total = (z - torch.where(torch.isinf(top), 0.0, top)).exp_().sum(-1, keepdim=True)
    return torch.where(total > 0, total.log(), -math.inf) + top


def _lse(s):
    z = _scores(s)
    return _normaliser(z).reshape(s["q"].shape[:3])


def _shared_plain(s):
    z = _scores(s)
    B, H, rep, L, S = z.shape
    lse = _normaliser(z)
    p = z.sub_(torch.where(torch.isinf(lse), 0.0, lse)).exp_()
    o = p.view(B, H, rep * L, S) @ _rows(s["cache"], "v", S)
    return [o.view(B, H * rep, L, -1).to(torch.bfloat16), lse.view(B, H * rep, L)]


def _weigh_plain(s):
    z = _scores(s)
    B, H, rep, L, S = z.shape
    lse = s["lse"].view(B, H, rep, L, 1)
    got = z.sub_(torch.where(torch.isinf(lse), 0.0, lse)).exp_().sum((2, 3))  # [B, H, S]
    row = torch.arange(S, device=z.device)
    fresh = (s["lens"] - s["rows"])[:, None]
    new = ((row >= fresh) & (row < s["lens"][:, None]))[:, None]
    w, p = s["weights"], s["positions"]
    # rows behind the last one stay (their sums are 0)
    w[:, :, :S] = torch.where(new, 0.0, w[:, :, :S]) + got
    at = (s["seen"] - s["rows"])[:, None] + (row - fresh)
    p[:, :, :S] = torch.where(new, at[:, None].int(), p[:, :, :S])
    return [w, p]


def _order(x):
    """Whole numbers in the order of float32 values, NaN below all."""
    bits = (x + 0.0).view(torch.int32).long()
    bits = torch.where(bits < 0, -2147483648 - bits, bits)
    return torch.where(torch.isnan(x), -(1 << 31), bits)


def _evict_plain(s):
    case, c = s["case"], s["cache"]
    keep, page = case["keep"], c["page"]
    w, p, table = s["weights"], s["positions"], c["table"]
    B, H, N = w.shape
    row = torch.arange(N, device=w.device)
    lens = s["lens"].long()[:, None, None]
    there = row < lens                                                        # [B, 1, N]
    newest = torch.where(there, p, -2147483648).amax(-1, keepdim=True).long()
    safe = (row < case["first"]) | (p.long() > newest - case["recent"])
    key = torch.where(safe, 1 << 31, _order(w))
    key = torch.where(there, key, -(1 << 32))
    best = torch.topk((key << 24) + (N - 1 - row), min(keep, N), dim=-1).indices
    kept = torch.zeros((B, H, N), dtype=torch.bool, device=w.device).scatter_(-1, best, True)
    kept = torch.where(lens > keep, kept, there)  # shorter ones stay whole
    hole = (row < keep) & there & ~kept
    tail = (row >= keep) & there & kept
    # the j-th hole takes the j-th kept row behind
    rank = torch.where(tail, tail.cumsum(-1) - 1, N)
    source = torch.zeros((B, H, N + 1), dtype=torch.long, device=w.device)
    source.scatter_(-1, rank, row.expand(B, H, N))
    at = (hole.cumsum(-1) - 1).clamp(min=0)
    M = min(N, -(-keep // page) * page)
    origin = torch.where(hole, source.gather(-1, at), row)[..., :M]           # [B, H, M]
    live = (there & (row < keep))[..., :M].expand(B, H, M)
    moved = (origin != row[:M]) & live
    ids = table.long()[:, None].expand(B, H, -1).gather(-1, origin // page)   # [B, H, M]
    to = table.long()[:, None].expand(B, H, -1).gather(-1, (row[:M] // page).expand(B, H, M))
    head = torch.arange(H, device=w.device)[None, :, None].expand(B, H, M)
    for name in ("k", "v"):
        codes, scales = c[name + "_codes"], c[name + "_scales"]
        was = scales[ids, head]                                               # [B, H, M]
        top = torch.where(live, was, 0.0).view(B, H, M // page, page).amax(-1)
        some = moved.view(B, H, M // page, page).any(-1)
        now = torch.where(some, top, scales[to, head].view(B, H, M // page, page)[..., 0])
        now = now.repeat_interleave(page, -1)
        ratio = torch.where(now > 0, was / now, 1.0)
        x = codes[ids, head, origin % page].float()
        x = torch.where(live[..., None], torch.round(x * ratio[..., None]),
                        codes[to, head, (row[:M] % page).expand(B, H, M)].float())
        # pages of sequences that are not touched may be in no table at all
        codes[to, head, (row[:M] % page).expand(B, H, M)] = x.to(torch.int8)
        scales[to, head] = now
    for t in (w, p):
        t[..., :M] = torch.where(moved, t.gather(-1, origin), t[..., :M])
    lens = s["lens"].clamp(max=keep)
    n = min(keep, N)
    inside = (row[:n] < lens[:, None])[:, None, :, None]
    read = [torch.where(inside, _rows(c, name, n)[:, :, :n], 0.0).to(torch.bfloat16)
            for name in ("k", "v")]
    return [lens, w, p, *read]


def _rotate_plain(s):
    case = s["case"]
    half = case["rope"] // 2
    axis = torch.tensor(s["axes"], device=s["q"].device)
    freq = ROPE_BASE ** (-torch.arange(half, device=axis.device, dtype=torch.float64) / half)
    angle = s["positions"].double()[axis].permute(1, 2, 0) * freq             # [B, L, half]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    got = []
    for name in ("q", "k"):
        x = s[name].float()
        if s[name + "_norm"] is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * s[name + "_norm"].float()
        a, b = x[..., :half], x[..., half:2 * half]
        x = torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]), -1)
        got.append(x.to(torch.bfloat16).contiguous())
    return got


def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        if op == "rotate":
            from vates_b200.rotary import rotate_axes
            return list(rotate_axes(s["q"], s["k"], s["positions"], s["axes"], base=ROPE_BASE,
                                    q_norm=s["q_norm"], k_norm=s["k_norm"]))
        cache = s["handle"]
        if op == "shared":
            return list(cache.attend_shared(s["q"], s["lens"], s["plan"], q_lens=s["rows"],
                                            return_lse=True))
        if op == "weigh":
            cache.weigh(s["q"], s["lse"], s["lens"], s["weights"], q_lens=s["rows"],
                        positions=s["positions"], seen=s["seen"])
            return [s["weights"], s["positions"]]
        lens = cache.evict(s["weights"], s["lens"], case["keep"], first=case["first"],
                           recent=case["recent"], positions=s["positions"])
        return [lens, s["weights"], s["positions"], *cache.read(lens, case["keep"])]
    if op == "rotate":
        return _rotate_plain(s)
    if op == "shared":
        return _shared_plain(s)
    return _weigh_plain(s) if op == "weigh" else _evict_plain(s)


# ------------------------------------------------------------ 64-bit results
def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "rotate":
        return _rotate_exact(s)
    lens = [(int(n), int(k)) for n, k in zip(s["rows"].tolist(), s["lens"].tolist())]
    if case["op"] == "evict":
        return _evict_exact(s, lens)
    c, page = s["cache"], case["page"]
    B, H, D, rep, L = case["batch"], case["kv_heads"], case["dim"], case["rep"], case["L"]
    table = c["table"].tolist()
    shared = case["op"] == "shared"
    if shared:
        out = torch.zeros((B, H * rep, L, D), dtype=torch.float64, device="cuda")
        lse = torch.full((B, H * rep, L), -math.inf, dtype=torch.float64, device="cuda")
    else:
        weights = s["weights"].double()
    for b, (n, keys) in enumerate(lens):
        if not n:
            continue
        ids = table[b][:-(-keys // page)]

        def values(name):
            x = c[name + "_codes"][ids].double() * c[name + "_scales"][ids].double()[..., None, None]
            return x.transpose(0, 1).reshape(H, -1, D)[:, :keys]

        k = values("k")
        v = values("v") if shared else None
        reach = torch.arange(n, device="cuda")[:, None] + (keys - n)
        hide = torch.arange(keys, device="cuda") > reach                      # [n, keys]
        for h in range(H):
            q = s["q"][b, h * rep:(h + 1) * rep, :n].double()                 # [rep, n, D]
            z = (q @ k[h].t() / math.sqrt(D)).masked_fill(hide, -math.inf)
            if shared:
                lse[b, h * rep:(h + 1) * rep, :n] = torch.logsumexp(z, -1)
                out[b, h * rep:(h + 1) * rep, :n] = torch.softmax(z, -1) @ v[h]
            else:
                p = torch.exp(z - s["lse"][b, h * rep:(h + 1) * rep, :n].double()[..., None])
                weights[b, h, keys - n:keys] = 0
                weights[b, h, :keys] += p.sum((0, 1))
    return [out, lse] if shared else [weights, None]


def _evict_exact(s, lens):
    case, c = s["case"], s["cache"]
    keep, page, H, D, B = case["keep"], case["page"], case["kv_heads"], case["dim"], case["batch"]
    weights = s["weights"].cpu()
    positions = s["positions"].cpu()
    table = c["table"].cpu()
    out = {n: torch.zeros((B, H, keep, D), dtype=torch.float64, device="cuda") for n in ("k", "v")}
    after = weights.double()
    for b, (_, n) in enumerate(lens):
        for h in range(H):
            order = list(range(n))
            w, at = weights[b, h, :n].tolist(), positions[b, h, :n].tolist()
            new = order
            if n > keep:
                late = max(at) - case["recent"]
                order.sort(key=lambda i: (not (i < case["first"] or at[i] > late),
                                          -w[i] if not (i < case["first"] or at[i] > late) else 0, i))
                kept = set(order[:keep])
                behind = iter(sorted(i for i in kept if i >= keep))
                new = [i if i in kept else next(behind) for i in range(keep)]
            if not new:
                continue
            idx = torch.tensor(new)
            after[b, h, :len(new)] = weights[b, h, idx].double()
            own_row = idx == torch.arange(len(new))
            ids, at_row = table[b, idx // page].long().cuda(), (idx % page).cuda()
            to = torch.arange(len(new)) // page
            for name in ("k", "v"):
                scale = c[name + "_scales"][ids, h].double().cpu()
                most = torch.zeros(int(to[-1]) + 1, dtype=torch.float64)
                most.scatter_reduce_(0, to, scale, "amax")
                touched = torch.zeros_like(most).scatter_reduce_(0, to, (~own_row).double(), "amax")
                now = torch.where(touched[to] > 0, most[to], scale)
                code = c[name + "_codes"][ids, h, at_row].double()
                ratio = torch.where(now > 0, scale / now, 1.0).cuda()
                out[name][b, h, :len(new)] = torch.round(code * ratio[:, None]) * now.cuda()[:, None]
    return [None, after, None, out["k"], out["v"]]


def _rotate_exact(s):
    case, got = s["case"], []
    half = case["rope"] // 2
    freq = torch.tensor([math.exp(-math.log(ROPE_BASE) * i / half) for i in range(half)],
                        dtype=torch.float64, device="cuda")
    turn = torch.stack([s["positions"][a] for a in s["axes"]], -1).double() * freq
    unit = torch.polar(torch.ones_like(turn), turn)[:, None]                  # [B, 1, L, half]
    for name in ("q", "k"):
        x = s[name].double()
        if s[name + "_norm"] is not None:
            x = x / torch.sqrt((x ** 2).mean(-1, keepdim=True) + 1e-6) * s[name + "_norm"].double()
        y = torch.complex(x[..., :half], x[..., half:2 * half]) * unit
        got.append(torch.cat((y.real, y.imag, x[..., 2 * half:]), -1))
    return got
