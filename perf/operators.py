"""Operators of a paged compressed cache, as cases that can be timed and compared.

The pages of a serving program's pool hold keys and values as this framework compresses them: packed code rows (codeword index and
radius code per chunk of four values), a scale per token and, with outlier extraction, flag words and the original values of the
flagged chunks.  Three operators work on the pages of a ragged batch:

  attend  ``paged_attention``: the last tokens of every sequence (one, a few, or a prompt chunk) attend over the sequence's pages,
          causally, with an optional sliding window, a cap on the scores (cap * tanh(score / cap)) and a sink logit per head
  mass    ``paged_attention_mass``: the softmax weight that every cached token receives from those queries, summed over the query
          heads of its KV head and over the queries, on top of a decayed earlier sum
  evict   ``paged_evict``: per sequence and KV head the first and the last tokens and the heaviest of the others move, in order, to
          the pages of a smaller table; the kept places and weights come with them

``own`` False: elementary torch operations in 32 bits.  ``own`` True: the framework's calls on the same planes."""
import math
import random

import torch

own = False

HEADS = ((32, 8, 128), (28, 4, 128), (64, 8, 64))        # query heads, KV heads, head dim
CODEBOOKS = ((24, 3), (96, 4), (192, 6))                  # secondary codebook size, radius bits
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
# outlier channels (chunk columns) per head, and the share of other chunks that are outliers: of the keys, of the values
OUTLIERS = {"none": ((0, 0.0), (0, 0.0)), "hot": ((2, 0.002), (0, 0.002)), "spiky": ((0, 0.005), (0, 0.005)), "onehot": ((1, 0.001), (1, 0.001))}


def _case(kind, name=None, *, heads=0, book=1, B=1, T=1024, q=1, page=64, out="none", window=0, cap=0.0, sinks=False, dtype="bf16", keep=0):
    c = {} if name is None else {"name": name}
    Hq, Hkv, d = HEADS[heads]
    S, rb = CODEBOOKS[book]
    c.update(kind=kind, Hq=Hq, Hkv=Hkv, d=d, S=S, rb=rb, B=B, T=T, q=q, page=page, out=out, window=window, cap=cap, sinks=sinks,
             dtype=dtype, keep=keep)
    return c


def listed():
    return [
        # one user's next token over a short context: a call whose launches count
        _case("attend", "attend_1x1013", book=0, T=1013, dtype="fp16"),
        # the decode step of a serving batch at long, ragged contexts; outlier channels in the keys
        _case("attend", "attend_16x32k", B=16, T=32768, out="hot"),
        # head dim 64, eight query heads per KV head, a sink logit per head, an outlier channel in every head
        _case("attend", "attend_64x8k_d64_sinks", heads=2, B=64, T=8192, out="onehot", sinks=True),
        # four drafted tokens of every sequence are verified at once; seven query heads per KV head, 19-bit fields
        _case("attend", "attend_8x8111_verify", heads=1, book=2, B=8, T=8111, q=4, out="spiky", page=128),
        # chunked prefill: up to 500 new tokens of four prompts
        _case("attend", "attend_4x8k_chunk_500", B=4, T=8192, q=500, out="hot"),
        # a long prompt's last chunk, scores capped
        _case("attend", "attend_1x16k_chunk_2k_cap", T=16384, q=2048, cap=30.0, out="hot"),
        # weights of one decode step, short and long
        _case("mass", "mass_1x2000", book=0, T=2000),
        _case("mass", "mass_16x16k", B=16, T=16384, out="hot"),
        # the weights that the last 32 tokens of a prompt give: what to keep of it
        _case("mass", "mass_4x8k_last_32", B=4, T=8192, q=32, out="spiky"),
        # prompts cut down to a budget before decoding: short ones, a serving batch, one very long document
        _case("evict", "evict_2x1000_to_256", B=2, T=1000, keep=256, out="hot"),
        _case("evict", "evict_16x8k_to_2k", B=16, T=8192, keep=2048, out="hot"),
        _case("evict", "evict_1x128k_to_16k", book=2, T=131072, keep=16384, out="spiky", page=128),
    ]


def _log_int(rng, lo, hi):
    hi = max(lo, int(hi))
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(("attend", "attend", "attend", "mass", "mass", "evict", "evict"))
    heads = rng.randrange(len(HEADS))
    book = rng.randrange(len(CODEBOOKS)) if heads < 2 else 1
    out = rng.choice(("none", "hot", "spiky", "onehot"))
    c = dict(heads=heads, book=book, out=out, page=rng.choice((64, 64, 128, 256)), dtype=rng.choice(("bf16", "bf16", "fp16")))
    Hq, Hkv, d = HEADS[heads]
    row = Hkv * d
    if kind == "evict":
        c["B"] = _log_int(rng, 1, 32)
        c["T"] = _log_int(rng, 100, min(131072, 130_000_000 // (c["B"] * row)))
        c["keep"] = _log_int(rng, 32, c["T"])
        return _case(kind, **c)
    c["window"] = rng.choice((0, 0, 0, 128, 1000))
    c["cap"] = rng.choice((0.0, 0.0, 30.0, 50.0))
    c["sinks"] = rng.random() < 0.3
    if kind == "mass":
        c["B"] = _log_int(rng, 1, 32)
        c["q"] = rng.choice((1, 1, _log_int(rng, 2, 64)))
        c["T"] = _log_int(rng, max(64, c["q"]), min(32768, 260_000_000 // (c["B"] * row), 500_000_000 // (c["B"] * Hq * c["q"])))
        return _case(kind, **c)
    how = rng.choice(("token", "token", "few", "chunk"))
    if how == "token":
        c["B"] = _log_int(rng, 1, 64)
        c["T"] = _log_int(rng, 20, min(131072, 500_000_000 // (c["B"] * row)))
        return _case(kind, **c)
    c["q"] = _log_int(rng, 2, 16) if how == "few" else _log_int(rng, 17, 2048)
    c["B"] = _log_int(rng, 1, 32 if how == "few" else 4)
    c["T"] = _log_int(rng, c["q"], min(32768, 260_000_000 // (c["B"] * row), 1_000_000_000 // (c["B"] * Hq * c["q"])))
    return _case(kind, **c)


# ---- what a case consists of --------------------------------------------------------------------------------------------------
def _lengths(c):
    """Tokens held and new tokens of every sequence: the longest first, the others down to half of it."""
    T, q = c["T"], c["q"]
    kv = [T - (i * 7919) % max(1, T // 2) if i else T for i in range(c["B"])]
    new = [max(1, q - (i * 37) % max(1, q // 2)) if q > 4 else q for i in range(c["B"])]
    return kv, [min(n, k) for n, k in zip(new, kv)]


def _index_bits(S):
    return math.ceil(math.log2(24 * S))


def _qmul(a, b):
    aw, ax, ay, az = a.unbind(-1)
    bw, bx, by, bz = b.unbind(-1)
    return torch.stack([aw * bw - ax * bx - ay * by - az * bz, aw * bx + ax * bw + ay * bz - az * by,
                        aw * by - ax * bz + ay * bw + az * bx, aw * bz + ax * by - ay * bx + az * bw], -1)


def _table(H, S, gen):
    """Codewords of every head in the cache's index order ((a * S + s) * 8 + unit): axis unit times omega^a times secondary s."""
    axis = torch.eye(4, device="cuda").repeat_interleave(2, 0) * torch.tensor([1.0, -1.0], device="cuda").repeat(4).unsqueeze(1)
    omega = torch.full((4,), 0.5, device="cuda")
    power = torch.stack([torch.tensor([1.0, 0, 0, 0], device="cuda"), omega, _qmul(omega, omega)])
    q = torch.nn.functional.normalize(torch.randn(H, S, 4, generator=gen, device="cuda"), dim=-1)
    first = _qmul(axis.view(1, 8, 4), power.view(3, 1, 4))                                           # [3][8]
    return _qmul(first.view(1, 3, 1, 8, 4), q.view(H, 1, S, 1, 4)).reshape(H, 24 * S, 4).half().contiguous()


def _planes(c, n_pages, channels, share, gen):
    """The planes of one tensor's pages: codes, scales and, with outliers, flags, block offsets, values and counts."""
    H, pt, N, S, rb = c["Hkv"], c["page"], c["d"] // 4, c["S"], c["rb"]
    dt, ib = DTYPES[c["dtype"]], _index_bits(c["S"])
    rows = (n_pages, H, pt)
    norm = torch.randn(*rows, N, 4, generator=gen, device="cuda").square_().sum(-1).sqrt_()
    flag = None
    if c["out"] != "none":
        at = torch.rand(H, N, generator=gen, device="cuda").argsort(1)[:, :channels]
        hot = torch.zeros(H, N, device="cuda").scatter_(1, at, 1.0).bool().view(1, H, 1, N).expand(*rows, N)
        flag = hot | (torch.rand(*rows, N, generator=gen, device="cuda") < share)
        norm = torch.where(flag, norm.clamp_(min=1.0) * 8.0, norm)
    rs = norm.amax(-1).to(dt)
    qmax = (1 << rb) - 1
    rq = (norm * (qmax / rs.float()).unsqueeze(-1)).round_().clamp_(0, qmax).to(torch.int32)
    if flag is not None:
        rq.masked_fill_(flag, 0)
    field = torch.randint(0, 24 * S, rq.shape, generator=gen, device="cuda", dtype=torch.int32) | (rq << ib)
    del rq
    words = (N * (ib + rb) + 31) // 32
    packed = torch.zeros(*rows, words + 1, dtype=torch.int64, device="cuda")
    for k in range(N):
        bit = k * (ib + rb)
        v = field[..., k].to(torch.int64) << (bit & 31)
        packed[..., bit >> 5] |= v & 0xffffffff
        packed[..., (bit >> 5) + 1] |= v >> 32
    packed = packed[..., :words]
    p = {"codes": torch.where(packed >= 1 << 31, packed - (1 << 32), packed).to(torch.int32).view(torch.uint8), "rs": rs}
    if flag is not None:
        per = flag.sum(-1).view(n_pages, H, pt // 16, 16).sum(-1)
        off = torch.zeros(n_pages, H, pt // 16 + 1, dtype=torch.int32, device="cuda")
        off[..., 1:] = per.cumsum(-1)
        cap = (int(pt * (channels + 4 * share * N) + 40) + 1) & ~1
        vals = torch.zeros(n_pages, H, cap, 4, dtype=dt, device="cuda")
        hit = flag.view(n_pages, H, pt * N)
        a, b, e = hit.nonzero(as_tuple=True)
        place = (hit.cumsum(-1, dtype=torch.int32) - 1)[a, b, e].long()
        x = torch.nn.functional.normalize(torch.randn(len(a), 4, generator=gen, device="cuda"), dim=-1) * norm.view(n_pages, H, pt * N)[a, b, e].unsqueeze(1)
        room = place < cap
        vals[a[room], b[room], place[room]] = x[room].to(dt)
        p["flags"] = (flag.to(torch.int64) << torch.arange(N, device="cuda")).sum(-1)
        p["flags"] = torch.where(p["flags"] >= 1 << 31, p["flags"] - (1 << 32), p["flags"]).to(torch.int32)
        p.update(out_off=off, out_vals=vals, out_count=off[..., -1].contiguous())
    return p


def _state(c, seed):
    """Inputs of a case: planes, tables of pages, queries or weights."""
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    kv, new = _lengths(c)
    pt, dt = c["page"], DTYPES[c["dtype"]]
    kept = [min(c["keep"], n) for n in kv] if c["kind"] == "evict" else []
    need = [-(-n // pt) for n in kv + kept]
    n_pages = sum(need) + 3
    order = list(range(n_pages))
    random.Random(int(seed)).shuffle(order)
    tables, at = [], 0
    for n in need:
        tables.append(order[at:at + n])
        at += n
    wide = max(len(t) for t in tables)
    s = {"case": c, "kv": kv, "new": new, "kept": kept, "tables": tables[:len(kv)], "new_tables": tables[len(kv):]}
    s["pages"] = torch.tensor([t + [0] * (wide - len(t)) for t in tables], device="cuda")
    s["kv_lens"], s["q_lens"] = torch.tensor(kv, device="cuda"), torch.tensor(new, device="cuda")
    s["kept_lens"] = torch.tensor(kept, device="cuda")
    s["table_K"], s["table_V"] = _table(c["Hkv"], c["S"], gen), _table(c["Hkv"], c["S"], gen)
    (ck, sk), (cv, sv) = OUTLIERS[c["out"]]
    s["K"] = _planes(c, n_pages, ck, sk, gen)
    if c["kind"] != "mass":
        s["V"] = _planes(c, n_pages, cv, sv, gen)
    if c["kind"] == "evict":
        # accumulated weights: a few heavy tokens, many light ones, some that no query has looked at
        w = torch.empty(n_pages, c["Hkv"], pt, device="cuda").exponential_(1.0, generator=gen).pow_(3)
        s["mass"] = torch.where(torch.rand(w.shape, generator=gen, device="cuda") < 0.1, torch.zeros_like(w), w)
        s["new_mass"] = torch.zeros_like(s["mass"])
        for x in (s["K"], s["V"]):                       # the pages to be filled are fresh
            free = torch.tensor(sum(s["new_tables"], []), device="cuda")
            for name, t in x.items():
                t[free] = 0
    else:
        s["Q"] = (1.5 * torch.randn(sum(new), c["Hq"], c["d"], generator=gen, device="cuda")).to(dt)
        s["sinks"] = torch.randn(c["Hq"], generator=gen, device="cuda") + 1.0 if c["sinks"] else None
    if c["kind"] == "mass":
        s["prior"] = torch.empty(n_pages, c["Hkv"], pt, device="cuda").exponential_(1.0, generator=gen)
        s["mass"] = torch.zeros_like(s["prior"])
    s["n_pages"] = n_pages
    return s


def prepare(case, seed):
    s = _state(case, seed)
    if own:
        _handles(s)
    return s


def _handles(s):
    """The framework's objects for the same planes: the pool, and the batch with its plan."""
    import hqmq_b200 as hqmq
    c = s["case"]
    cap = s["K"]["out_vals"].shape[2] if c["out"] != "none" else None
    cap_v = s["V"]["out_vals"].shape[2] if c["out"] != "none" and "V" in s else cap
    dt = DTYPES[c["dtype"]]
    s["pool"] = hqmq.PagedKV(s["n_pages"], c["Hkv"], c["d"], c["S"], c["rb"], "cuda", page_tokens=c["page"], dtype=dt,
                             outliers_K=c["out"] != "none", outliers_V=c["out"] != "none", out_cap=(cap, cap_v))
    for side in ("K", "V"):
        for name, t in s.pop(side, {}).items():
            getattr(s["pool"], side).pages(name).copy_(t)
    s["batch"] = hqmq.PagedBatch(s["pool"], s["tables"], s["kv"], s["new"], n_heads=c["Hq"], window=c["window"] or None)
    if c["kind"] == "evict":
        s["target"] = hqmq.PagedBatch(s["pool"], s["new_tables"], s["kept"])


# ---- plain forms ----------------------------------------------------------------------------------------------------------------
def _outlier_entries(p):
    """(flagged [page, H, token, chunk], place of every chunk's entry among its page's)."""
    N = p["n"]
    bits = (p["flags"].unsqueeze(-1) >> torch.arange(N, device="cuda")) & 1
    return bits.bool(), bits.view(*bits.shape[:2], -1).cumsum(-1).view(bits.shape) - bits


def _values(c, p, table, pages):
    """Dense fp32 values [B, H, tokens, d] of the pages named in `pages` [B, n]."""
    N, S, rb, ib = c["d"] // 4, c["S"], c["rb"], _index_bits(c["S"])
    words = p["codes"].view(torch.int32)[pages].to(torch.int64) & 0xffffffff                       # [B, n, H, pt, words]
    words = torch.cat([words, torch.zeros_like(words[..., :1])], -1)
    bit = torch.arange(N, device="cuda") * (ib + rb)
    field = ((words[..., bit >> 5] | (words[..., (bit >> 5) + 1] << 32)) >> (bit & 31)) & ((1 << (ib + rb)) - 1)
    del words
    at = (field & ((1 << ib) - 1)) + (torch.arange(c["Hkv"], device="cuda") * 24 * S).view(1, 1, -1, 1, 1)
    rs = p["rs"][pages].float()
    x = table.view(-1, 4)[at].float() * ((field >> ib) * (rs / ((1 << rb) - 1)).unsqueeze(-1)).unsqueeze(-1)
    del field, at
    if "flags" in p:
        flagged, place = _outlier_entries({**p, "flags": p["flags"][pages].flatten(0, 1), "n": N})
        flagged, place = flagged.view(*x.shape[:-1]), place.view(*x.shape[:-1])
        cap = p["out_vals"].shape[2]
        first = (pages.unsqueeze(-1) * c["Hkv"] + torch.arange(c["Hkv"], device="cuda")).view(*pages.shape, -1, 1, 1) * cap
        v = p["out_vals"].view(-1, 4)[first + place.clamp(max=cap - 1)].float() * (place < cap).unsqueeze(-1)
        x = torch.where(flagged.unsqueeze(-1), v, x)
    B, n, H, pt = x.shape[:4]
    return x.permute(0, 2, 1, 3, 4, 5).reshape(B, H, n * pt, 4 * N)


def _padded(s, wide):
    """Queries [B, H_q, wide, d] and their places [B, wide] in the ragged tensor, with what is no query at place 0."""
    first = s["q_lens"].cumsum(0) - s["q_lens"]
    i = torch.arange(wide, device="cuda")
    real = i < s["q_lens"].unsqueeze(1)
    place = torch.where(real, first.unsqueeze(1) + i, 0)
    return s["Q"].float()[place].permute(0, 2, 1, 3), place, real


def _scores(s, K, wide):
    """Masked scores [B, H_kv, G * wide, T] of the padded queries."""
    c = s["case"]
    G = c["Hq"] // c["Hkv"]
    q, place, real = _padded(s, wide)
    B, T = q.shape[0], K.shape[2]
    x = (q.reshape(B, c["Hkv"], G * wide, c["d"]) @ K.transpose(-1, -2)).mul_(1.0 / math.sqrt(c["d"])).view(B, c["Hkv"], G, wide, T)
    if c["cap"]:
        x = torch.tanh(x / c["cap"]) * c["cap"]
    t, pos = torch.arange(T, device="cuda"), (s["kv_lens"] - s["q_lens"]).unsqueeze(1) + torch.arange(wide, device="cuda")
    see = (t <= pos.unsqueeze(-1)) & real.unsqueeze(-1)                                              # [B, wide, T]
    if c["window"]:
        see &= t > pos.unsqueeze(-1) - c["window"]
    return x.masked_fill_(~see.view(B, 1, 1, wide, T), -math.inf), place, real


def _weights(s, x):
    """exp(score - largest) in place of the scores, and one over their sum (with the sinks); rows that see nothing give zeros."""
    c = s["case"]
    m = x.amax(-1, keepdim=True)
    if s["sinks"] is not None:
        sink = s["sinks"].view(1, c["Hkv"], -1, 1, 1)
        m = torch.maximum(m, sink)
    m = torch.where(m == -math.inf, 0.0, m)
    p = x.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    if s["sinks"] is not None:
        total = total + (sink - m).exp()
    return p, torch.where(total > 0, 1.0 / total, 0.0)


def _attend(s):
    c, wide = s["case"], max(s["new"])
    K = _values(c, s["K"], s["table_K"], s["pages"])
    x, place, real = _scores(s, K, wide)
    del K
    p, inv = _weights(s, x)
    V = _values(c, s["V"], s["table_V"], s["pages"])
    # (what is behind a sequence's last token has no weight, whatever its page holds)
    V = V.masked_fill_((torch.arange(V.shape[2], device="cuda") >= s["kv_lens"].unsqueeze(1)).view(V.shape[0], 1, -1, 1), 0.0)
    B = V.shape[0]
    o = (p.flatten(2, 3) @ V).view(B, c["Hkv"], -1, wide, c["d"]) * inv
    o = o.permute(0, 3, 1, 2, 4).reshape(B, wide, c["Hq"], c["d"])
    return o[real].to(s["Q"].dtype)


def _mass(s):
    c, wide = s["case"], max(s["new"])
    x, place, real = _scores(s, _values(c, s["K"], s["table_K"], s["pages"]), wide)
    p, inv = _weights(s, x)
    w = p.mul_(inv).sum((2, 3))                                                                     # [B, H_kv, T]
    B, pt = w.shape[0], c["page"]
    w = w.view(B, c["Hkv"], -1, pt).transpose(1, 2)
    live = (torch.arange(w.shape[1] * pt, device="cuda").view(-1, pt) < s["kv_lens"].view(-1, 1, 1)).unsqueeze(2).expand_as(w)
    at = s["pages"].view(B, -1, 1, 1)
    h, t = torch.arange(c["Hkv"], device="cuda").view(1, 1, -1, 1), torch.arange(pt, device="cuda")
    at, h, t = (y.expand_as(w)[live] for y in (at, h, t))
    s["mass"][at, h, t] = 0.75 * s["prior"][at, h, t] + w[live]
    return s["mass"]


SINK_TOKENS, RECENT_TOKENS = 4, 16


def _evict(s):
    c, pt = s["case"], s["case"]["page"]
    B, H, N = c["B"], c["Hkv"], c["d"] // 4
    src, dst = s["pages"][:B], s["pages"][B:, :max(len(t) for t in s["new_tables"])]
    kv, kept = s["kv_lens"].view(B, 1, 1), s["kept_lens"].view(B, 1, 1)
    mass = s["mass"][src].transpose(1, 2).flatten(2)                                                # [B, H, T]
    t = torch.arange(mass.shape[2], device="cuda").expand_as(mass)
    # the last tokens first, then the first ones, then by weight; of equal ones the earlier
    rank = torch.where(t >= kv, -math.inf, torch.where(t >= kv - RECENT_TOKENS, math.inf, torch.where(t < SINK_TOKENS, 3e38, mass)))
    order = rank.argsort(dim=-1, descending=True, stable=True)
    n_max = max(s["kept"])
    i = torch.arange(n_max, device="cuda").expand(B, H, n_max)
    chosen = torch.where(i < kept, order[..., :n_max], 1 << 30).sort(-1).values
    real = i < kept
    chosen = torch.where(real, chosen, 0)
    b, h = torch.arange(B, device="cuda").view(-1, 1, 1).expand_as(i)[real], torch.arange(H, device="cuda").view(1, -1, 1).expand_as(i)[real]
    frm, to = chosen[real], i[real]
    sp, st, dp, dt = src[b, frm // pt], frm % pt, dst[b, to // pt], to % pt
    for p in (s["K"], s["V"]):
        p["codes"][dp, h, dt] = p["codes"][sp, h, st]
        p["rs"][dp, h, dt] = p["rs"][sp, h, st]
        if "flags" in p:
            cap = p["out_vals"].shape[2]
            p["flags"][dp, h, dt] = p["flags"][sp, h, st]
            used = torch.unique(dp)
            # (behind a sequence's last token no flag counts)
            bits_d, place_d = _outlier_entries({"flags": p["flags"][used], "n": N})
            count = torch.zeros(len(used), H, pt, dtype=torch.int32, device="cuda")
            where = torch.searchsorted(used, dp)
            live = torch.zeros(len(used), H, pt, dtype=torch.bool, device="cuda")
            live[where, h, dt] = True
            count[live] = bits_d.sum(-1, dtype=torch.int32)[live]
            off = torch.zeros(len(used), H, pt // 16 + 1, dtype=torch.int32, device="cuda")
            off[..., 1:] = count.view(len(used), H, -1, 16).sum(-1).cumsum(-1)
            p["out_off"][used] = off
            p["out_count"][used] = off[..., -1]
            bits_s, place_s = _outlier_entries({"flags": p["flags"], "n": N})
            k, ch = bits_s[sp, h, st].nonzero(as_tuple=True)
            a, z = place_s[sp[k], h[k], st[k], ch], place_d[where[k], h[k], dt[k], ch]
            k, a, z = k[z < cap], a[z < cap], z[z < cap]
            x = p["out_vals"][sp[k], h[k], a.clamp(max=cap - 1)]
            p["out_vals"][dp[k], h[k], z] = torch.where((a < cap).unsqueeze(1), x, torch.zeros_like(x))
    s["new_mass"][dp, h, dt] = s["mass"][sp, h, st]
    return {"kept": torch.where(real, chosen, -1).to(torch.int32), "mass": s["new_mass"], "K": dict(s["K"]), "V": dict(s["V"])}


def run(s):
    c = s["case"]
    if own:
        import hqmq_b200 as hqmq
        more = {} if c["kind"] == "evict" else {"softcap": c["cap"] or None, "sinks": s["sinks"]}
        if c["kind"] == "attend":
            return hqmq.paged_attention(s["Q"], s["pool"], s["batch"], s["table_K"], s["table_V"], **more)
        if c["kind"] == "mass":
            return hqmq.paged_attention_mass(s["Q"], s["pool"], s["batch"], s["table_K"], prior=s["prior"], decay=0.75, out=s["mass"], **more)
        kept = hqmq.paged_evict(s["pool"], s["batch"], s["target"], s["mass"], first=SINK_TOKENS, last=RECENT_TOKENS, out_mass=s["new_mass"])
        return {"kept": kept, "mass": s["new_mass"], "K": s["pool"].K.planes(), "V": s["pool"].V.planes()}
    return {"attend": _attend, "mass": _mass, "evict": _evict}[c["kind"]](s)


# ---- bytes and operations ---------------------------------------------------------------------------------------------------------
def _token_bytes(c, side):
    """Compressed bytes of one token of one KV head, keys (0) or values (1)."""
    N = c["d"] // 4
    n = N * (_index_bits(c["S"]) + c["rb"]) / 8 + 2
    if c["out"] != "none":
        channels, share = OUTLIERS[c["out"]][side]
        n += N / 8 + 8 * (channels + (N - channels) * share)
    return n


def work(case):
    c = case
    kv, new = _lengths(c)
    Hq, Hkv, d = c["Hq"], c["Hkv"], c["d"]
    both = _token_bytes(c, 0) + _token_bytes(c, 1)
    if c["kind"] == "evict":
        kept = sum(min(c["keep"], n) for n in kv)
        # every weight is read once, the kept rows and weights are read and written
        return {"bytes": Hkv * (4 * sum(kv) + kept * (2 * both + 8)), "flops": Hkv * sum(kv)}
    w = c["window"]
    keys = sum(min(n, w + q - 1) if w else n for n, q in zip(kv, new))
    pairs = sum(sum(min(n - q + i + 1, w or n) for i in range(q)) for n, q in zip(kv, new))
    rows = sum(new) * Hq * d
    if c["kind"] == "attend":
        return {"bytes": Hkv * keys * both + 4 * rows, "flops": 4 * Hq * d * pairs}
    return {"bytes": Hkv * (keys * _token_bytes(c, 0) + 8 * sum(kv)) + 2 * rows, "flops": 2 * Hq * d * pairs}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------------------
def _dense64(c, p, table, pages, length):
    """[H, length, d] in 64 bits of one sequence: token after token of its pages, decoded from the definition."""
    N, ib, H = c["d"] // 4, _index_bits(c["S"]), c["Hkv"]
    codes = torch.cat([p["codes"][i] for i in pages], 1)[:, :length]                                # [H, T, row bytes]
    bits = ((codes.unsqueeze(-1) >> torch.arange(8, device="cuda", dtype=torch.uint8)) & 1).flatten(-2)[..., :N * (ib + c["rb"])]
    bits = bits.view(H, length, N, ib + c["rb"])
    idx = sum(bits[..., k].long() << k for k in range(ib))
    rq = sum(bits[..., ib + k].double() * 2 ** k for k in range(c["rb"]))
    rs = torch.cat([p["rs"][i] for i in pages], 1)[:, :length].double()
    x = torch.stack([table[h].double()[idx[h]] for h in range(H)]) * (rq * rs.unsqueeze(-1) / ((1 << c["rb"]) - 1)).unsqueeze(-1)
    if "flags" in p:
        for k, page in enumerate(pages):
            fl = ((p["flags"][page].unsqueeze(-1) >> torch.arange(N, device="cuda")) & 1).bool()    # [H, pt, N]
            h, t, ch = fl.nonzero(as_tuple=True)                                                    # head by head, token by token
            entry = torch.arange(len(h), device="cuda") - torch.searchsorted(h, h)                  # (a head's entries count from 0)
            cap, ok = p["out_vals"].shape[2], t < length - k * c["page"]
            v = p["out_vals"][page, h, entry.clamp(max=cap - 1)].double() * (entry < cap).unsqueeze(1)
            x[h[ok], k * c["page"] + t[ok], ch[ok]] = v[ok]
    return x.reshape(H, length, c["d"])


def exact(case, seed):
    c = case
    s = _state(c, seed)
    if c["kind"] == "evict":
        kept = torch.full((c["B"], c["Hkv"], max(s["kept"])), -1, dtype=torch.int32)
        mass, new_mass = s["mass"].cpu(), s["new_mass"].cpu().double()
        for b in range(c["B"]):
            w = torch.cat([mass[i] for i in s["tables"][b]], 1)[:, :s["kv"][b]]
            for h in range(c["Hkv"]):
                n, k = s["kv"][b], s["kept"][b]
                row = w[h].tolist()
                first = [(0 if t >= n - RECENT_TOKENS else 1 if t < SINK_TOKENS else 2, -row[t], t) for t in range(n)]
                first = [x if x[0] else (0, 0.0, x[2]) for x in first]
                first = [x if x[0] != 1 else (1, 0.0, x[2]) for x in first]
                got = sorted(t for _, _, t in sorted(first)[:k])
                kept[b, h, :k] = torch.tensor(got, dtype=torch.int32)
                for i, t in enumerate(got):
                    new_mass[s["new_tables"][b][i // c["page"]], h, i % c["page"]] = row[t]
        return {"kept": kept, "mass": new_mass, "K": None, "V": None}
    G = c["Hq"] // c["Hkv"]
    outs, mass, first = [], None, 0
    if c["kind"] == "mass":
        mass = s["mass"].double()
    for b, (T, n) in enumerate(zip(s["kv"], s["new"])):
        k = _dense64(c, s["K"], s["table_K"], s["tables"][b], T)
        v = _dense64(c, s["V"], s["table_V"], s["tables"][b], T) if c["kind"] == "attend" else None
        q = s["Q"][first:first + n].double().view(n, c["Hkv"], G, c["d"]).permute(1, 2, 0, 3)
        first += n
        sc = torch.einsum("hgid,htd->hgit", q, k) / math.sqrt(c["d"])
        if c["cap"]:
            sc = c["cap"] * torch.tanh(sc / c["cap"])
        i, t = torch.arange(n, device="cuda").view(n, 1) + T - n, torch.arange(T, device="cuda")
        sc = sc.masked_fill(~((t <= i) & (t > i - (c["window"] or T + 1))), -math.inf)
        if c["sinks"]:
            sc = torch.cat([sc, s["sinks"].double().view(c["Hkv"], G, 1, 1).expand(-1, -1, n, 1)], -1)
        w = torch.softmax(sc, -1)[..., :T]
        if c["kind"] == "attend":
            outs.append(torch.einsum("hgit,htd->ihgd", w, v).reshape(n, c["Hq"], c["d"]))
        else:
            total = w.sum((1, 2))
            for k_, page in enumerate(s["tables"][b]):
                m = min(c["page"], T - k_ * c["page"])
                mass[page, :, :m] = 0.75 * s["prior"][page, :, :m].double() + total[:, k_ * c["page"]:k_ * c["page"] + m]
    return torch.cat(outs) if c["kind"] == "attend" else mass
