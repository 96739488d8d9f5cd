"""Cases for the 8-bit paged KV cache and the token log probabilities.

Four operators: writing key/value rows into a paged cache of int8 codes with
one scale per page and key/value head ("write", returned as the values that
the touched pages then stand for), reading rows back ("read"), attention over
the cache ("attend"), and log probabilities of given tokens with rank,
entropy and the best alternatives ("logprob").

The cache (one layer): codes int8 ``[pages, Hkv, page, D]``, scales float32
``[pages, Hkv]`` for K and for V, and a table int32 ``[B, max_pages]`` with
the pool page of every ``page`` consecutive positions of a sequence.
"""
import math
import random

import torch

own = False

VOCAB = 151936      # vocabulary of the decode stack
MIN_SCALE = 2.0 ** -40


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # one decode step of one sequence through the decode stack's attention layer
        dict(name="write_one", op="write", batch=1, n=1, kv_heads=2, dim=256, page=64, pos=1000,
             ragged=False),
        # a verify step (up to 4 rows each) of a batch of sequences at odd positions
        dict(name="write_verify", op="write", batch=24, n=4, kv_heads=8, dim=128, page=32,
             pos=3001, ragged=True),
        # two long prompts written at once behind a short shared prefix
        dict(name="write_prompt", op="write", batch=2, n=65536, kv_heads=2, dim=256, page=64,
             pos=75, ragged=False),
        # the last rows of a few sequences, moved to another cache
        dict(name="read_tail", op="read", batch=3, n=301, kv_heads=4, dim=64, page=16, pos=515,
             ragged=True),
        # a whole 131,072-token sequence
        dict(name="read_long", op="read", batch=1, n=131072, kv_heads=2, dim=256, page=64, pos=0,
             ragged=False),
        # a decode step early in an answer
        dict(name="attend_one", op="attend", batch=1, L=1, kv_heads=2, rep=8, dim=256, page=64,
             keys=901, ragged=False, causal=True),
        # a verify step of a batch of sequences of mixed lengths, some slots idle
        dict(name="attend_verify", op="attend", batch=16, L=4, kv_heads=8, rep=4, dim=128, page=32,
             keys=8190, ragged=True, causal=True),
        # a decode step at the end of a 131,072-token context
        dict(name="attend_long", op="attend", batch=1, L=1, kv_heads=2, rep=8, dim=256, page=64,
             keys=131072, ragged=False, causal=True),
        # prompts of mixed odd lengths, five query heads to a key/value head, small heads
        dict(name="prefill_ragged", op="attend", batch=3, L=733, kv_heads=4, rep=5, dim=64,
             page=16, keys=1467, ragged=True, causal=True),
        # one 4096-row chunk of a long prompt
        dict(name="prefill_long", op="attend", batch=1, L=4096, kv_heads=2, rep=8, dim=256,
             page=64, keys=32768, ragged=False, causal=True),
        # the rows of one verify step
        dict(name="logprob_step", op="logprob", rows=4, vocab=VOCAB, top=5, dtype="bfloat16",
             temperature=1.0, banned=0.0),
        # scoring the tokens of a prompt
        dict(name="logprob_prompt", op="logprob", rows=2048, vocab=VOCAB, top=20,
             dtype="bfloat16", temperature=1.0, banned=0.0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("write", "read", "attend", "attend", "prefill", "logprob"))
    if op == "logprob":
        vocab = _log_int(rng, 1000, 200000) | 1 if rng.random() < 0.5 else VOCAB
        rows = _log_int(rng, 1, max(1, 2048 * VOCAB // vocab // 2))
        return dict(op=op, rows=min(rows, 4096), vocab=vocab, top=rng.choice((0, 1, 5, 20, 32)),
                    dtype=rng.choice(("bfloat16", "float32")),
                    temperature=rng.choice((1.0, 0.7, 1.3)), banned=rng.choice((0.0, 0.3)))
    base = dict(op=op, kv_heads=rng.choice((1, 2, 4, 8)), dim=rng.choice((64, 128, 256)),
                page=rng.choice((16, 32, 64, 128)), ragged=rng.random() < 0.6)
    width = base["kv_heads"] * base["dim"]
    if op in ("write", "read"):
        batch = _log_int(rng, 1, 32)
        most = max(1, 2 * 65536 * 512 // (width * batch))
        base.update(batch=batch, n=_log_int(rng, 1, min(131072, most)),
                    pos=_log_int(rng, 1, 5000) - 1)
        return base
    base.update(rep=rng.choice((1, 2, 3, 4, 5, 7, 8, 16)), causal=rng.random() < 0.8)
    if op == "attend":
        batch = _log_int(rng, 1, 32)
        L = rng.choice((1, 1, 1, 2, 3, 4, 5, 8))
        most = max(64, 131072 * 512 // (width * batch))
        base.update(batch=batch, L=L, keys=_log_int(rng, max(16, L), most))
        return base
    base.update(op="attend", batch=_log_int(rng, 1, 4), L=_log_int(rng, 16, 4096))
    heads = base["kv_heads"] * base["rep"] * base["batch"]
    pairs = 4096 * 32768 * 16 * 256 // (heads * base["dim"] * 2)
    most = max(base["L"], min(32768, pairs // base["L"], 131072 * 512 // (width * base["batch"])))
    base["keys"] = _log_int(rng, base["L"], most)
    return base


# --------------------------------------------------------- lengths of a case
def _lengths(case):
    """Per-sequence (rows of this pass, positions before them), from the case alone."""
    B = case["batch"]
    rows = case["n"] if case["op"] in ("write", "read") else case["L"]
    before = case["pos"] if case["op"] in ("write", "read") else max(0, case["keys"] - rows)
    r = random.Random(1000003 * rows + 101 * before + B)
    got = []
    for b in range(B):
        if not case["ragged"] or b == 0:
            got.append((rows, before))
        elif b % 8 == 5:
            got.append((0, 0))  # an idle slot of the batch
        else:
            got.append((r.randint(max(1, rows // 4), rows), int(before * r.uniform(0.05, 1.0))))
    return got


def _visible(case):
    """(query, key) pairs of one query head over the batch."""
    total = 0
    for n, before in _lengths(case):
        total += n * before + (n * (n + 1) // 2 if case["causal"] else n * n)
    return total


def work(case):
    if case["op"] == "logprob":
        size = 2 if case["dtype"] == "bfloat16" else 4
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * (16 + 8 * case["top"]), "flops": 5 * n}
    width = case["kv_heads"] * case["dim"]
    page = case["page"]
    lens = _lengths(case)
    if case["op"] == "write":
        new = sum(n for n, _ in lens)
        window = _window(case)
        # rows in (bf16), codes out, and the touched pages read back (codes in, bf16 out)
        seen = sum(p + n - p // page * page for n, p in lens if n)
        return {"bytes": 2 * width * (3 * new + seen + 2 * window * case["batch"]),
                "flops": 2 * width * 4 * new}
    if case["op"] == "read":
        seen = sum(n for n, _ in lens)
        return {"bytes": 2 * width * (seen + 2 * case["n"] * case["batch"]),
                "flops": 2 * width * seen}
    heads = case["kv_heads"] * case["rep"]
    keys = sum(n + p for n, p in lens if n)
    io = case["batch"] * heads * case["L"] * (4 * case["dim"] + 4)
    return {"bytes": 2 * width * keys + io, "flops": 4 * case["dim"] * heads * _visible(case)}


def _window(case):
    """Rows of the pages that a write of this case can touch, per sequence."""
    return ((case["n"] + case["page"] - 2) // case["page"] + 1) * case["page"]


# ------------------------------------------------------------------- inputs
def _cache(case, g, lens, device):
    """A cache with room for every sequence, its pages in shuffled order."""
    page, H, D, B = case["page"], case["kv_heads"], case["dim"], case["batch"]
    reach = _window(case) if case["op"] == "write" else page
    need = [(n + p) // page + 1 + (reach // page if n else 0) for n, p in lens]
    width = max(need)
    pages = B * width + 1  # the last page is in no table
    order = torch.randperm(B * width, generator=g, device=device)
    table = order.view(B, width).to(torch.int32)
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


def prepare(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    s = dict(case=case)
    if case["op"] == "logprob":
        R, V = case["rows"], case["vocab"]
        dtype = getattr(torch, case["dtype"])
        logits = torch.empty((R, V), dtype=dtype, device=device)
        step = max(1, (1 << 27) // V)
        for i in range(0, R, step):  # normal logits with a few likely tokens per row
            part = torch.randn((min(step, R - i), V), generator=g, device=device) * 2.5
            hot = torch.randint(0, V, (part.shape[0], 8), generator=g, device=device)
            lift = torch.rand(hot.shape, generator=g, device=device) * 10.0
            part.scatter_add_(1, hot, lift)
            if case["banned"]:  # constrained decoding: tokens that cannot follow
                part.masked_fill_(torch.rand(part.shape, generator=g, device=device)
                                  < case["banned"], -math.inf)
            logits[i:i + step] = part.to(dtype)
        tokens = torch.randint(0, V, (R,), generator=g, device=device)
        best = torch.empty(R, dtype=torch.int64, device=device)
        for i in range(0, R, step):
            best[i:i + step] = logits[i:i + step].float().argmax(-1)
        likely = torch.rand(R, generator=g, device=device) < 0.5
        s.update(logits=logits, tokens=torch.where(likely, best, tokens).to(torch.int32))
        if own:
            import vates_b200.logprobs  # noqa: F401
        return s
    lens = _lengths(case)
    s["cache"] = _cache(case, g, lens, device)
    rows = torch.tensor([n for n, _ in lens], dtype=torch.int32, device=device)
    pos = torch.tensor([p for _, p in lens], dtype=torch.int32, device=device)
    s.update(rows=rows, pos=pos, lens=rows + pos)
    B, H, D = case["batch"], case["kv_heads"], case["dim"]
    if case["op"] == "write":
        n = case["n"]
        for name in ("keys", "values"):  # channels of unequal size
            x = torch.randn((B, H, n, D), generator=g, device=device)
            x *= torch.rand((1, H, 1, D), generator=g, device=device) + 0.5
            s[name] = x.to(torch.bfloat16)
        s["start"] = torch.div(pos, case["page"], rounding_mode="floor").int() * case["page"]
        s["window"] = _window(case)
    elif case["op"] == "read":
        s["start"], s["window"] = pos, case["n"]
    else:
        q = torch.randn((B, H * case["rep"], case["L"], D), generator=g, device=device)
        s["q"] = (q * 1.5).to(torch.bfloat16)
    if own:
        from vates_b200.kv8 import PagedKV8Cache
        c = s["cache"]
        s["handle"] = PagedKV8Cache(c["k_codes"], c["v_codes"], c["k_scales"], c["v_scales"],
                                    c["table"])
    return s


# ---------------------------------------------------------------- plain form
def _touched(cache, start, window):
    """Pool pages of the rows [start, start + window) of each sequence; the
    page that is in no table past the end of the table."""
    page, table = cache["page"], cache["table"]
    idx = torch.div(start, page, rounding_mode="floor").long()[:, None] + \
        torch.arange(window // page, device=start.device)
    ids = table.long().gather(1, idx.clamp(max=table.shape[1] - 1))
    return torch.where(idx < table.shape[1], ids, cache["k_codes"].shape[0] - 1)


def _write_plain(s):
    c, page, W = s["cache"], s["cache"]["page"], s["window"]
    B, H, n, D = s["keys"].shape
    first = torch.div(s["pos"], page, rounding_mode="floor") * page
    position = first[:, None] + torch.arange(W, device=first.device)          # [B, W]
    row = position - s["pos"][:, None]
    new = (row >= 0) & (row < s["rows"][:, None])
    old = row < 0
    ids = _touched(c, first, W)                                               # [B, W/page]
    touched = new.view(B, -1, page).any(-1)
    ids = torch.where(touched, ids, c["k_codes"].shape[0] - 1)
    held = old.view(B, -1, page).any(-1)
    pick = row.clamp(0, n - 1).long()[:, None, :, None].expand(B, H, W, D)
    for src, name in (("keys", "k"), ("values", "v")):
        x = s[src].gather(2, pick).float()
        x = torch.where(new[:, None, :, None], x, 0.0).view(B, H, W // page, page, D)
        amax = x.abs().amax((-1, -2)).permute(0, 2, 1)                        # [B, W/page, H]
        scale = torch.where(amax > 0, (amax / 127.0).clamp(min=MIN_SCALE), 0.0)
        before = torch.where(held[..., None], c[name + "_scales"][ids], 0.0)
        scale = torch.maximum(scale, before)
        inv = torch.where(scale > 0, 1.0 / scale, 0.0)
        ratio = torch.where(scale > 0, before / scale, 1.0)                  # 1 where it stays
        codes = c[name + "_codes"][ids].float()                               # [B, P, H, page, D]
        kept = torch.round(codes * ratio[..., None, None])
        fresh = torch.round(x.permute(0, 2, 1, 3, 4) * inv[..., None, None]).clamp(-127, 127)
        is_new = new.view(B, W // page, 1, page, 1)
        is_old = old.view(B, W // page, 1, page, 1)
        out = torch.where(is_new, fresh, torch.where(is_old, kept, codes))
        c[name + "_codes"][ids] = out.to(torch.int8)
        c[name + "_scales"][ids] = torch.where(touched[..., None], scale, c[name + "_scales"][ids])
    return _read_plain(c, s["start"], W, s["lens"])


def _read_plain(c, start, n, lens):
    page, table = c["page"], c["table"]
    position = start[:, None].long() + torch.arange(n, device=start.device)   # [B, n]
    inside = position < lens[:, None]
    idx = torch.div(position, page, rounding_mode="floor").clamp(max=table.shape[1] - 1)
    ids, at = table.long().gather(1, idx), position % page
    got = []
    for name in ("k", "v"):
        x = c[name + "_codes"][ids, :, at].float() * c[name + "_scales"][ids][..., None]
        x = torch.where(inside[..., None, None], x, 0.0)
        got.append(x.permute(0, 2, 1, 3).to(torch.bfloat16))
    return got


def _attend_plain(s):
    case, c = s["case"], s["cache"]
    B, Hq, L, D = s["q"].shape
    H, rep, page = case["kv_heads"], case["rep"], c["page"]
    n_pages = -(-case["keys"] // page)
    ids = c["table"][:, :n_pages].long()
    S = n_pages * page

    def rows(name):
        x = c[name + "_codes"][ids].float() * c[name + "_scales"][ids][..., None, None]
        return x.permute(0, 2, 1, 3, 4).reshape(B, H, S, D)

    q = s["q"].float().view(B, H, rep * L, D)
    scores = (q @ rows("k").transpose(-1, -2)).mul_(D ** -0.5).view(B, H, rep, L, S)
    key = torch.arange(S, device=q.device)
    i = torch.arange(L, device=q.device)
    last = s["lens"][:, None].expand(B, L)
    if case["causal"]:
        last = (s["lens"] - s["rows"])[:, None] + i + 1
    last = torch.where(i < s["rows"][:, None], last, 0)                       # keys seen by row i
    hidden = key >= last[..., None]                                           # [B, L, S]
    scores.masked_fill_(hidden[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(torch.isinf(top), 0.0, top)).exp_()
    total = scores.sum(-1, keepdim=True)
    lse = (torch.where(total > 0, total.log(), -math.inf) + top)[..., 0]
    o = scores.view(B, H, rep * L, S) @ rows("v")
    o = o.view(B, H, rep, L, D) / torch.where(total > 0, total, 1.0)
    return [o.reshape(B, Hq, L, D).to(torch.bfloat16), lse.reshape(B, Hq, L)]


def _order(x, V):
    """Whole numbers in the order of (value, lower index first)."""
    bits = x.view(torch.int32)
    bits = torch.where(bits < 0, ~bits ^ -2147483648, bits).long()
    return (bits << 32) + (V - 1 - torch.arange(V, device=x.device))


def _logprob_plain(s):
    case = s["case"]
    x = s["logits"].float() + 0.0
    R, V = x.shape
    tok = s["tokens"].long()[:, None]
    key = _order(x, V)
    rank = (key > key.gather(1, tok)).sum(-1)
    best = torch.topk(key, case["top"], dim=-1).values if case["top"] else key[:, :0]
    ids = V - 1 - (best & 0xFFFFFFFF)
    del key
    top_x = x.gather(1, ids)
    tok_x = x.gather(1, tok)
    inv = 1.0 / case["temperature"]
    x.mul_(inv)
    top = x.amax(-1, keepdim=True)
    x.sub_(top)
    p = x.exp()
    total = p.sum(-1, keepdim=True)
    x.clamp_(min=-1000.0)
    entropy = total.log()[:, 0] - (p.mul_(x)).sum(-1) / total[:, 0]
    lse = total.log() + top
    return [(tok_x * inv - lse)[:, 0], rank.to(torch.int32), entropy,
            ids.to(torch.int32), top_x * inv - lse]


def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        if op == "logprob":
            from vates_b200.logprobs import token_logprobs
            return list(token_logprobs(s["logits"], s["tokens"], top=case["top"],
                                       temperature=case["temperature"]))
        cache = s["handle"]
        if op == "write":
            cache.append(s["keys"], s["values"], s["pos"], counts=s["rows"])
            return [*cache.read(s["lens"], s["window"], start=s["start"]),
                    cache.k_scales, cache.v_scales]
        if op == "read":
            return list(cache.read(s["lens"], s["window"], start=s["start"]))
        return list(cache.attend(s["q"], s["lens"], q_lens=s["rows"], causal=case["causal"],
                                 return_lse=True))
    if op == "logprob":
        return _logprob_plain(s)
    if op == "write":
        c = s["cache"]
        return [*_write_plain(s), c["k_scales"], c["v_scales"]]
    if op == "read":
        return _read_plain(s["cache"], s["start"], s["window"], s["lens"])
    return _attend_plain(s)


# ------------------------------------------------------------ 64-bit results
def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "logprob":
        return _logprob_exact(s)
    lens = [(int(n), int(p)) for n, p in zip(s["rows"].tolist(), s["pos"].tolist())]
    c, page = s["cache"], case["page"]
    B, H, D = case["batch"], case["kv_heads"], case["dim"]
    table = c["table"].tolist()

    def values(name, b, lo, hi):
        """float64 rows [lo, hi) of sequence b, [H, hi - lo, D]."""
        first, last = lo // page, -(-hi // page)
        ids = table[b][first:last]
        x = c[name + "_codes"][ids].double() * c[name + "_scales"][ids].double()[..., None, None]
        return x.transpose(0, 1).reshape(H, -1, D)[:, lo - first * page:hi - first * page]

    if case["op"] == "write":
        W = s["window"]
        outs = []
        for src, name in (("keys", "k"), ("values", "v")):
            scales = c[name + "_scales"].double()
            out = torch.zeros((B, H, W, D), dtype=torch.float64, device="cuda")
            for b, (n, p) in enumerate(lens):
                if not n:
                    continue
                head = p - p // page * page
                top = -(-(head + n) // page)
                ids = table[b][p // page:p // page + top]
                x = torch.zeros((H, top * page, D), dtype=torch.float64, device="cuda")
                x[:, head:head + n] = s[src][b, :, :n].double()
                x = x.view(H, top, page, D)
                sc = x.abs().amax((-1, -2)) / 127
                sc = torch.where(sc > 0, sc.clamp(min=MIN_SCALE), sc)
                was = scales[ids].t()
                if head:
                    sc[:, 0] = torch.maximum(sc[:, 0], was[:, 0])
                q = torch.round(x / torch.where(sc > 0, sc, 1.0)[..., None, None]).clamp(-127, 127)
                if head:
                    old = c[name + "_codes"][ids[0]][:, :head].double()
                    q[:, 0, :head] = torch.round(old * (was[:, 0] / sc[:, 0])[:, None, None])
                scales[ids] = sc.t()
                out[b, :, :head + n] = (q * sc[..., None, None]).reshape(H, -1, D)[:, :head + n]
            outs.append((out, scales))
        return [outs[0][0], outs[1][0], outs[0][1], outs[1][1]]
    if case["op"] == "read":
        outs = []
        for name in ("k", "v"):
            out = torch.zeros((B, H, case["n"], D), dtype=torch.float64, device="cuda")
            for b, (n, p) in enumerate(lens):
                out[b, :, :n] = values(name, b, p, p + n)
            outs.append(out)
        return outs
    rep, L = case["rep"], case["L"]
    out = torch.zeros((B, H * rep, L, D), dtype=torch.float64, device="cuda")
    lse = torch.full((B, H * rep, L), -math.inf, dtype=torch.float64, device="cuda")
    for b, (n, p) in enumerate(lens):
        if not n:
            continue
        k, v = values("k", b, 0, n + p), values("v", b, 0, n + p)
        step = max(1, (1 << 28) // (n + p))
        for h in range(H * rep):
            for i in range(0, n, step):
                q = s["q"][b, h, i:min(n, i + step)].double()
                z = q @ k[h // rep].t() / math.sqrt(D)
                if case["causal"]:
                    at = torch.arange(i, i + len(q), device="cuda")[:, None] + p
                    z = z.masked_fill(torch.arange(n + p, device="cuda") > at, -math.inf)
                lse[b, h, i:i + len(q)] = torch.logsumexp(z, -1)
                out[b, h, i:i + len(q)] = torch.softmax(z, -1) @ v[h // rep]
    return [out, lse]


def _logprob_exact(s):
    case = s["case"]
    logits, R, k = s["logits"], case["rows"], case["top"]
    lp = torch.empty(R, dtype=torch.float64, device="cuda")
    ent, tops = torch.empty_like(lp), torch.empty((R, k), dtype=torch.float64, device="cuda")
    step = max(1, (1 << 26) // case["vocab"])
    for i in range(0, R, step):
        z = torch.log_softmax(logits[i:i + step].double() / case["temperature"], -1)
        lp[i:i + step] = z.gather(1, s["tokens"][i:i + step].long()[:, None])[:, 0]
        ent[i:i + step] = torch.special.entr(z.exp()).sum(-1)
        tops[i:i + step] = torch.sort(z, -1, descending=True).values[:, :k]
    return [lp, None, ent, None, tops]
