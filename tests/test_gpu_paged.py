"""Operators over a paged compressed cache against plain 64-bit implementations on the pages' own contents."""
import math
import random

import numpy as np
import pytest
import torch

import hqmq_b200 as hqmq
from hqmq_b200 import _lib
from hqmq_b200.packed import PackedKV

from .util import make_kv

pytestmark = pytest.mark.gpu
DEV = "cuda"


# ---- plain implementations ------------------------------------------------------------------------------------------------------
def dense64(planes, table, S, rb, pages, length):
    """(H, length, d) in 64 bits from page planes on the host, decoded bit by bit."""
    codes = torch.cat([planes["codes"][p] for p in pages], 1)[:, :length].numpy()
    H, _, N = codes.shape[0], length, planes["n"]
    ib = hqmq.packed.idx_bits(S)
    bits = np.unpackbits(codes, axis=-1, bitorder="little")[..., :N * (ib + rb)].reshape(H, length, N, ib + rb).astype(np.int64)
    idx = (bits[..., :ib] << np.arange(ib)).sum(-1)
    rq = (bits[..., ib:] << np.arange(rb)).sum(-1)
    rs = torch.cat([planes["rs"][p] for p in pages], 1)[:, :length].double().numpy()
    tab = table.double().cpu().numpy()
    x = np.stack([tab[h][idx[h]] for h in range(H)]) * (rq * rs[..., None] / ((1 << rb) - 1))[..., None]
    if "flags" in planes:
        T = planes["codes"].shape[2]
        for h in range(H):
            for k, p in enumerate(pages):
                e = 0
                for t in range(min(T, length - k * T)):
                    word = int(planes["flags"][p, h, t]) & 0xffffffff
                    for c in range(N):
                        if word >> c & 1:
                            cap = planes["out_vals"].shape[2]
                            x[h, k * T + t, c] = planes["out_vals"][p, h, e].double().numpy() if e < cap else 0.0
                            e += 1
    return torch.from_numpy(x.reshape(H, length, 4 * N))


def host(pk):
    return {**{k: v.cpu() for k, v in pk.planes().items()}, "n": pk.n_chunks}


def attend64(q, k, v, G, window, cap, sinks, scale):
    """Outputs (q, H_q, d), weights (H_kv, keys) and bounds of what operands in 11 bits can be off, of one sequence."""
    n, Hq, d = q.shape
    T = k.shape[1]
    qq = q.double().view(n, Hq // G, G, d).permute(1, 2, 0, 3)                       # H_kv, G, n, d
    s = torch.einsum("hgid,htd->hgit", qq, k) * scale
    size = torch.einsum("hgid,htd->hgit", qq.abs(), k.abs()) * abs(scale)
    if cap:
        s = cap * torch.tanh(s / cap)
    pos, t = torch.arange(n).view(n, 1) + T - n, torch.arange(T)
    see = (t <= pos) & (t > pos - (window or T + 1))
    s = s.masked_fill(~see, -math.inf)
    if sinks is not None:
        s = torch.cat([s, sinks.double().view(-1, G, 1, 1).expand(-1, -1, n, 1)], -1)
    p = torch.softmax(s, -1)[..., :T]
    o = torch.einsum("hgit,htd->ihgd", p, v).reshape(n, Hq, d)
    # A key's values reach the product with 11 bits (2^-11 relative), so a score is off by at most 2^-11 of the sum of its products' sizes,
    # a weight by that and the weights' mean of it; values by 2^-11, weights by 2^-11 (rounding) and 2^-25 of 2^0..2^1
    # times the largest (fp16's smallest step, whose size V's scales can double)
    e = 2.0 ** -11
    off = size * see * e
    rel = off + (p * off).sum(-1, keepdim=True)
    va = v.abs()
    bound = torch.einsum("hgit,htd->ihgd", p * (rel + 3 * e), va) + T * 2.0 ** -24 * va.amax()
    return o, p.sum((1, 2)), bound.reshape(n, Hq, d), (p * (rel / e) * 2.0 ** -20).sum((1, 2))


HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


class World:
    """A pool filled through the encoder and paged_store, in several rounds of appends; other content where no token is."""

    def __init__(self, H, d, S, rb, kv, *, page=64, outliers="both", dtype=torch.bfloat16, rounds=3, seed=0, spare=4, out_cap=None,
                 garbage=True, kind="spiky"):
        rng = random.Random(seed)
        self.H, self.d, self.S, self.rb, self.kv, self.dtype, self.page = H, d, S, rb, kv, dtype, page
        need = [-(-n // page) for n in kv]
        self.n_pages = sum(need) + spare
        order = list(range(self.n_pages))
        rng.shuffle(order)
        self.tables, at = [], 0
        for n in need:
            self.tables.append(order[at:at + n])
            at += n
        self.free = order[at:]
        q = hqmq.HQMQ(1, H, S, rb, device=DEV)
        self.inner, self.quant = q, hqmq.with_outlier_extraction(q, C=outliers if isinstance(outliers, float) else 3.0) if outliers else q
        self.pool = hqmq.PagedKV(self.n_pages, H, d, S, rb, DEV, page_tokens=page, dtype=dtype, outliers_K=bool(outliers),
                                 outliers_V=bool(outliers), out_cap=page * d // 4 if out_cap is None else out_cap)
        if garbage:        # recycled pages: rows, scales that are no number, flags, offsets and counts of an earlier life
            g = torch.Generator(device=DEV).manual_seed(seed)
            for pk in (self.pool.K, self.pool.V):
                for name, t in pk.planes().items():
                    if name == "codes":
                        t.random_(0, 256, generator=g)
                    elif t.is_floating_point():
                        t.fill_(float("nan"))
                    else:
                        t.random_(0, 1 << 20, generator=g)
        self.tab = [q.tables(0, i, DEV)["table16"] for i in (0, 1)]
        self.stored = [[], []]                    # per append: staging planes and which tokens
        held = [0] * len(kv)
        for r in range(rounds):
            new = [n - h if r == rounds - 1 else rng.randint(0, n - h) for n, h in zip(kv, held)]
            held = [h + m for h, m in zip(held, new)]
            if not sum(new):
                continue
            x = [make_kv(kind, (1, H, sum(new), d), seed + 10 * r + i, dtype).to(DEV) for i in (0, 1)]
            pair = [self.inner.new_cache(1, sum(new), d, DEV, scale_dtype=dtype, with_outliers=bool(outliers), out_dtype=dtype) for _ in (0, 1)]
            self.quant.encode_pair(*x, 0, *pair)
            hqmq.paged_store(self.pool, *pair, hqmq.PagedBatch(self.pool, [t[:-(-h // page)] for t, h in zip(self.tables, held)], held, new))
            self.stored[0].append((pair, list(held), new))

    def dense(self):
        if not hasattr(self, "_dense"):
            pk = [host(self.pool.K), host(self.pool.V)]
            self._dense = [[dense64(x, t, self.S, self.rb, pages, n) for pages, n in zip(self.tables, self.kv)] for x, t in zip(pk, self.tab)]
        return self._dense

    def batch(self, q_lens, G, window=None, **kw):
        return hqmq.PagedBatch(self.pool, self.tables, self.kv, q_lens, n_heads=self.H * G, window=window, **kw)


def queries(w, q_lens, G, dtype, seed=1, scale=1.5):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(sum(q_lens), w.H * G, w.d, generator=g)).to(dtype)


def check_attend(w, out, q, q_lens, G, window=None, cap=None, sinks=None, scale=None):
    scale = w.d ** -0.5 if scale is None else scale
    K, V = w.dense()
    at, out = 0, out.cpu()
    for s, n in enumerate(q_lens):
        if n:
            o, _, bound, _ = attend64(q[at:at + n], K[s], V[s], G, window, cap, None if sinks is None else sinks.cpu(), scale)
            # (fp32 sums and exponentials: 2^-18 of what is summed)
            limit = bound + o.abs() * (HALF[out.dtype] + 2.0 ** -18) + 1e-7
            off = (out[at:at + n].double() - o).abs()
            assert bool((off <= limit).all()), (s, float((off / limit).max()), float(off.max()))
        at += n


# ---- store ------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("H,d,S,rb,page,outliers,dtype", [
    (2, 128, 96, 4, 64, "both", torch.bfloat16), (3, 64, 24, 3, 128, "both", torch.float16), (1, 128, 192, 6, 256, None, torch.bfloat16),
    (2, 64, 48, 5, 64, "both", torch.bfloat16),
])
def test_store_moves_rows_flags_and_values(H, d, S, rb, page, outliers, dtype):
    w = World(H, d, S, rb, [1, 130, 64, 700, 15], page=page, outliers=outliers, dtype=dtype, rounds=4)
    planes = [host(w.pool.K), host(w.pool.V)]
    for pair, held, new in w.stored[0]:
        for side in (0, 1):
            src, dst = pair[side], planes[side]
            idx, rq, rs, fl = (None if x is None else x.cpu() for x in src.to_reference(0, sum(new)))
            rows = src.codes[:H * src.T_cap * src.row_bytes].view(H, src.T_cap, src.row_bytes).cpu()
            at = 0
            for s, (n, m) in enumerate(zip(held, new)):
                for t in range(n - m, n):
                    p, r = w.tables[s][t // page], t % page
                    assert torch.equal(dst["codes"][p, :, r], rows[:, at])
                    assert torch.equal(dst["rs"][p, :, r].float(), rs[0, :, at])
                    if outliers:
                        word = (fl[0, :, at].long() << torch.arange(d // 4)).sum(-1)
                        assert torch.equal(dst["flags"][p, :, r].long() & 0xffffffff, word)
                    at += 1
    if outliers:
        # every page's entries are its tokens' in order, and the offsets count them
        for side in (0, 1):
            dst = planes[side]
            for s, n in enumerate(w.kv):
                for k, p in enumerate(w.tables[s]):
                    m = min(page, n - k * page)
                    count = torch.tensor([[bin(int(x) & 0xffffffff).count("1") for x in dst["flags"][p, h, :m]] for h in range(H)])
                    assert torch.equal(dst["out_count"][p].long(), count.sum(1))
                    for b in range(-(-m // 16) + 1):
                        assert torch.equal(dst["out_off"][p, :, b].long(), count[:, :16 * b].sum(1))
        # and the values are the originals of the flagged chunks
        K = w.dense()[0]
        dec = [w.quant.decode(pair[0], 0, 0, dtype=torch.float32, T=sum(new)).cpu() for pair, _, new in w.stored[0]]
        for (pair, held, new), x in zip(w.stored[0], dec):
            at = 0
            for s, (n, m) in enumerate(zip(held, new)):
                a, b = K[s][:, n - m:n], x[0, :, at:at + m].double()
                assert float((a - b).abs().max() if m else 0.0) <= float(b.abs().max() if m else 0.0) * 2.0 ** -10
                at += m


def test_store_over_a_full_side_buffer_counts_and_drops():
    w = World(2, 128, 24, 3, [200, 70], out_cap=4, kind="hot")
    for pk in (w.pool.K, w.pool.V):
        n = pk.pages("out_count")[[p for t in w.tables for p in t]]
        assert int(n.max()) > 4
    with pytest.raises(_lib.HqmqError):
        w.pool.check()
    q = queries(w, [1, 40], 4, torch.bfloat16)
    out = hqmq.paged_attention(q.to(DEV), w.pool, w.batch([1, 40], 4), *w.tab)
    check_attend(w, out, q, [1, 40], 4)


# ---- attention ------------------------------------------------------------------------------------------------------------------------
FORMS = [(2, 4, 128, 96, 4), (1, 7, 128, 192, 6), (2, 8, 64, 96, 4), (3, 1, 128, 24, 3), (1, 16, 64, 24, 3), (2, 5, 128, 48, 5), (1, 3, 64, 192, 6), (1, 4, 64, 160, 4), (1, 2, 128, 256, 6)]


@pytest.mark.parametrize("H,G,d,S,rb", FORMS)
@pytest.mark.parametrize("q_lens,window,cap,sink", [
    ([1, 1, 1, 1, 1], None, None, False), ([1, 0, 1, 1, 2], 1, None, True), ([1, 2, 1, 2, 0], 100, 3.0, False),
    ([1, 100, 33, 1, 20], None, None, True), ([0, 200, 1, 300, 20], 70, 5.0, True),
])
def test_attention_of_ragged_batches(H, G, d, S, rb, q_lens, window, cap, sink):
    kv = [1, 230, 64, 777, 33]
    w = World(H, d, S, rb, kv, seed=H + G)
    dtype = torch.bfloat16 if G % 2 else torch.float16
    q = queries(w, q_lens, G, dtype)
    sinks = torch.randn(H * G, generator=torch.Generator().manual_seed(3)).to(DEV) if sink else None
    out = hqmq.paged_attention(q.to(DEV), w.pool, w.batch(q_lens, G, window), *w.tab, softcap=cap, sinks=sinks)
    assert out.dtype == dtype
    check_attend(w, out, q, q_lens, G, window, cap, sinks)


@pytest.mark.parametrize("page,outliers", [(64, None), (256, "both"), (1024, "both")])
@pytest.mark.parametrize("n_q", [1, 3, 60])
def test_attention_at_every_length_around_tiles_and_pages(page, outliers, n_q):
    kv = [n for n in (1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255, 257, 300) if n >= n_q]
    w = World(1, 64, 24, 3, kv, page=page, outliers=outliers)
    q = queries(w, [n_q] * len(kv), 4, torch.float16)
    out = hqmq.paged_attention(q.to(DEV), w.pool, w.batch([n_q] * len(kv), 4), *w.tab)
    check_attend(w, out, q, [n_q] * len(kv), 4)


@pytest.mark.parametrize("q_dtype,o_dtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.float32, torch.float16)])
def test_attention_types_strides_and_scale(q_dtype, o_dtype):
    q_lens = [1, 3, 50]
    w = World(2, 128, 96, 4, [90, 300, 160])
    # queries of every second head and token of a larger tensor, at an odd offset; the output likewise
    big = torch.zeros(2 * sum(q_lens), 2 * 8 + 1, 128 + 3, dtype=q_dtype)
    q = queries(w, q_lens, 4, torch.bfloat16).to(q_dtype)
    big[::2, 1::2, 1:129] = q
    view = big.to(DEV)[::2, 1::2, 1:129]
    out = torch.full((2 * sum(q_lens), 9, 129), 7.0, dtype=o_dtype, device=DEV)
    hqmq.paged_attention(view, w.pool, w.batch(q_lens, 4), *w.tab, softmax_scale=0.03, out=out[1::2, 1:, 1:])
    check_attend(w, out[1::2, 1:, 1:], q, q_lens, 4, scale=0.03)
    assert bool((out[::2] == 7).all() and (out[:, 0] == 7).all() and (out[:, :, 0] == 7).all())
    # heads that lie apart (a transposed tensor)
    t = q.permute(1, 0, 2).contiguous().to(DEV).permute(1, 0, 2)
    again = hqmq.paged_attention(t, w.pool, w.batch(q_lens, 4), *w.tab, softmax_scale=0.03)
    check_attend(w, again, q, q_lens, 4, scale=0.03)


@pytest.mark.parametrize("n_q", [1, 8, 40])
@pytest.mark.parametrize("q_pow,k_pow,v_pow", [(60, -60, -40), (-30, 30, 40), (20, -20, 0)])
def test_attention_of_values_far_from_one(n_q, q_pow, k_pow, v_pow):
    """Keys, values and queries whose sizes fp16 does not hold: operands are relative to powers of two."""
    w = World(1, 128, 96, 4, [200, 90], outliers="both")
    for pk, e in ((w.pool.K, k_pow), (w.pool.V, v_pow)):
        for name in ("rs", "out_vals"):
            pk.pages(name).mul_(2.0 ** e)
    q = (queries(w, [n_q, n_q], 4, torch.bfloat16).float() * 2.0 ** q_pow).to(torch.bfloat16)
    out = hqmq.paged_attention(q.to(DEV), w.pool, w.batch([n_q, n_q], 4), *w.tab).cpu()
    K, V = w.dense()
    for s in range(2):
        o, _, bound, _ = attend64(q[s * n_q:(s + 1) * n_q], K[s], V[s], 4, None, None, None, 128 ** -0.5)
        off = (out[s * n_q:(s + 1) * n_q].double() - o).abs()
        assert bool((off <= bound + o.abs() * (2.0 ** -8 + 2.0 ** -18)).all())


@pytest.mark.parametrize("cap", [0.01, 1.0, 30.0, 1e4])
def test_caps_from_small_to_large(cap):
    w = World(1, 128, 96, 4, [300, 70])
    for q_lens in ([1, 1], [40, 20]):
        q = queries(w, q_lens, 4, torch.bfloat16, scale=3.0)
        out = hqmq.paged_attention(q.to(DEV), w.pool, w.batch(q_lens, 4), *w.tab, softcap=cap)
        check_attend(w, out, q, q_lens, 4, cap=cap)


def test_a_shared_prefix_and_the_same_page_twice():
    w = World(2, 64, 24, 3, [200, 64])
    tables, kv, q_lens = [w.tables[0], w.tables[0][:2] + w.tables[1], w.tables[1] * 3], [200, 190, 192], [1, 1, 30]
    q = queries(w, q_lens, 4, torch.bfloat16)
    out = hqmq.paged_attention(q.to(DEV), w.pool, hqmq.PagedBatch(w.pool, tables, kv, q_lens, n_heads=8), *w.tab)
    w.tables, w.kv = tables, kv
    w.__dict__.pop("_dense", None)
    check_attend(w, out, q, q_lens, 4)
    with pytest.raises(ValueError):
        hqmq.paged_attention_mass(q.to(DEV), w.pool, hqmq.PagedBatch(w.pool, tables, kv, q_lens, n_heads=8), w.tab[0])


@pytest.mark.parametrize("plane", ["K", "V"])
def test_a_scale_that_is_no_number_shows(plane):
    w = World(1, 128, 24, 3, [300, 300, 100])
    getattr(w.pool, plane).pages("rs")[w.tables[1][1], 0, 7] = float("nan")
    for q_lens in ([1, 1, 1], [1, 30, 30]):
        q = queries(w, q_lens, 4, torch.bfloat16)
        out = hqmq.paged_attention(q.to(DEV), w.pool, w.batch(q_lens, 4), *w.tab).float()
        a, b = q_lens[0], q_lens[0] + q_lens[1]
        assert bool(out[a:b].isnan().all()) and not bool(out[:a].isnan().any()) and not bool(out[b:].isnan().any())


def test_pages_behind_four_gigabytes():
    """Rows, side buffers and offsets whose places pass 32 bits (K's codes are 4.6 GB)."""
    H, n_pages, kv = 8, 140_000, [700, 90]
    q = hqmq.HQMQ(1, H, 96, 4, device=DEV)
    quant = hqmq.with_outlier_extraction(q, C=3.0)
    pool = hqmq.PagedKV(n_pages, H, 128, 96, 4, DEV, outliers_K=True, outliers_V=True, out_cap=128)
    order = list(range(n_pages - 40, n_pages))
    random.Random(0).shuffle(order)
    tables, at = [], 0
    for n in kv:
        tables.append(order[at:at + -(-n // 64)])
        at += -(-n // 64)
    x = [make_kv("spiky", (1, H, sum(kv), 128), i, torch.bfloat16).to(DEV) for i in (0, 1)]
    pair = [quant.encode(x[i], 0, i) for i in (0, 1)]
    batch = hqmq.PagedBatch(pool, tables, kv, kv)
    hqmq.paged_store(pool, *pair, batch)
    tab = [q.tables(0, i, DEV)["table16"] for i in (0, 1)]
    used = [p for t in tables for p in t]
    planes = []
    for pk in (pool.K, pool.V):                  # (the used pages alone, as if they were a pool)
        planes.append({**{k: v[torch.tensor(used, device=DEV)].cpu() for k, v in pk.planes().items()}, "n": 32})
    local = [[used.index(p) for p in t] for t in tables]
    K, V = ([dense64(x_, t, 96, 4, pages, n) for pages, n in zip(local, kv)] for x_, t in zip(planes, tab))
    for q_lens in ([1, 1], [40, 90]):
        qq = torch.randn(sum(q_lens), 32, 128, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
        b = hqmq.PagedBatch(pool, tables, kv, q_lens, n_heads=32)
        out, a = hqmq.paged_attention(qq.to(DEV), pool, b, *tab).cpu(), 0
        for s, n in enumerate(q_lens):
            o, _, bound, _ = attend64(qq[a:a + n], K[s], V[s], 4, None, None, None, 128 ** -0.5)
            assert bool(((out[a:a + n].double() - o).abs() <= bound + o.abs() * (2.0 ** -8 + 2.0 ** -18) + 1e-7).all())
            a += n
    mass = hqmq.paged_attention_mass(qq.to(DEV), pool, b, tab[0])
    assert abs(float(mass.sum()) - 130 * 32) < 0.1
    dst = [order[at:at + 2], order[at + 2:at + 3]]
    kept = hqmq.paged_evict(pool, batch, hqmq.PagedBatch(pool, dst, [100, 50]), mass).cpu()
    for s, n in enumerate([100, 50]):
        for h in range(H):
            rows = [pool.K.pages("codes")[tables[s][t // 64], h, t % 64] for t in kept[s, h, :n].tolist()]
            assert torch.equal(torch.stack(rows), torch.cat([pool.K.pages("codes")[p, h] for p in dst[s]])[:n])


@pytest.mark.parametrize("d,S,rb", [(128, 96, 4), (64, 96, 4), (128, 192, 6), (128, 24, 3), (128, 128, 4)])
@pytest.mark.parametrize("C", [0.7, 1.1, 1.5])
def test_tiles_full_of_outliers(d, S, rb, C):
    """Far more flagged chunks in a tile than are staged, or have table entries: up to all of them, in K and V."""
    w = World(1, d, S, rb, [300, 90, 17], rounds=1, outliers=C, kind="randn")
    for q_lens in ([1, 1, 1], [8, 3, 1], [40, 90, 17]):
        q = queries(w, q_lens, 4, torch.bfloat16)
        check_attend(w, hqmq.paged_attention(q.to(DEV), w.pool, w.batch(q_lens, 4), *w.tab), q, q_lens, 4)
    q = queries(w, [1, 5, 1], 4, torch.bfloat16)
    mass = hqmq.paged_attention_mass(q.to(DEV), w.pool, w.batch([1, 5, 1], 4), w.tab[0])
    K, V = w.dense()
    _, m, _, bound = attend64(q[1:6], K[1], V[1], 4, None, None, None, d ** -0.5)
    got = torch.cat([mass[p] for p in w.tables[1]], 1)[:, :90].cpu().double()
    assert bool(((got - m).abs() <= bound + m * (2.0 ** -20 + 20 * 2.0 ** -24)).all())


def test_sinks_of_any_type_and_size():
    w = World(2, 128, 96, 4, [300, 90])
    for q_lens in ([1, 1], [40, 90]):
        q = queries(w, q_lens, 4, torch.bfloat16)
        sinks = torch.tensor([0.0, -float("inf"), 80.0, -80.0, 3.0, 1e4, -1e4, 1.5]).to(torch.bfloat16)
        out = hqmq.paged_attention(q.to(DEV), w.pool, w.batch(q_lens, 4), *w.tab, sinks=sinks.to(DEV))
        check_attend(w, out, q, q_lens, 4, sinks=sinks)
        assert bool((out[:, 5] == 0).all())
        off = hqmq.paged_attention(q.to(DEV), w.pool, w.batch(q_lens, 4), *w.tab, sinks=torch.full((8,), float("inf"), device=DEV))
        assert bool((off == 0).all())


def test_many_sequences_and_more_heads_than_sms():
    kv = [1 + (37 * i) % 150 for i in range(300)]
    w = World(2, 64, 24, 3, kv, rounds=2)
    q = queries(w, [1] * 300, 2, torch.bfloat16)
    check_attend(w, hqmq.paged_attention(q.to(DEV), w.pool, w.batch([1] * 300, 2, 40), *w.tab), q, [1] * 300, 2, 40)
    w = World(160, 64, 24, 3, [70, 20], rounds=1, outliers=None)
    q = queries(w, [1, 17], 1, torch.bfloat16)
    check_attend(w, hqmq.paged_attention(q.to(DEV), w.pool, w.batch([1, 17], 1), *w.tab), q, [1, 17], 1)


def test_a_long_sequence_is_cut_over_all_ctas():
    kv = [20000, 300]
    w = World(2, 64, 96, 4, kv, rounds=2, kind="randn", outliers=None)
    for q_lens in ([1, 1], [2, 2], [20, 1]):
        q = queries(w, q_lens, 8, torch.bfloat16)
        check_attend(w, hqmq.paged_attention(q.to(DEV), w.pool, w.batch(q_lens, 8), *w.tab), q, q_lens, 8)


def test_the_same_call_gives_the_same_bits():
    w = World(2, 128, 96, 4, [900, 77, 2000])
    q = queries(w, [1, 2, 60], 4, torch.bfloat16).to(DEV)
    b = w.batch([1, 2, 60], 4)
    first = hqmq.paged_attention(q, w.pool, b, *w.tab)
    mass = hqmq.paged_attention_mass(q, w.pool, b, w.tab[0])
    for _ in range(3):
        assert torch.equal(first, hqmq.paged_attention(q, w.pool, b, *w.tab))
        assert torch.equal(mass, hqmq.paged_attention_mass(q, w.pool, b, w.tab[0]))


# ---- weights ----------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("H,G,d,S,rb", FORMS)
@pytest.mark.parametrize("q_lens,window,cap,sink", [
    ([1, 1, 1, 1, 1], None, None, False), ([1, 0, 3, 40, 2], 100, 3.0, True), ([0, 2, 60, 1, 33], None, None, True),
])
def test_mass_of_ragged_batches(H, G, d, S, rb, q_lens, window, cap, sink):
    w = World(H, d, S, rb, [1, 230, 64, 777, 33], seed=H + G)
    dtype = torch.bfloat16 if G % 2 else torch.float16
    q = queries(w, q_lens, G, dtype)
    sinks = torch.randn(H * G, generator=torch.Generator().manual_seed(3)).to(DEV) if sink else None
    g = torch.Generator(device=DEV).manual_seed(4)
    prior = torch.rand(w.n_pages, H, w.page, device=DEV, generator=g)
    out = torch.full_like(prior, -5.0)
    hqmq.paged_attention_mass(q.to(DEV), w.pool, w.batch(q_lens, G, window), w.tab[0], softcap=cap, sinks=sinks, prior=prior, decay=0.5, out=out)
    K, V = w.dense()
    out, prior, at = out.cpu(), prior.cpu().double(), 0
    seen = torch.zeros(out.shape, dtype=torch.bool)
    for s, n in enumerate(q_lens):
        T = w.kv[s]
        if n:
            _, m, _, bound = attend64(q[at:at + n], K[s], V[s], G, window, cap, None if sinks is None else sinks.cpu(), d ** -0.5)
        else:
            m = bound = torch.zeros(H, T, dtype=torch.float64)
        at += n
        got = torch.cat([out[p] for p in w.tables[s]], 1)[:, :T].double()
        was = torch.cat([prior[p] for p in w.tables[s]], 1)[:, :T]
        for k, p in enumerate(w.tables[s]):
            seen[p, :, :min(w.page, T - k * w.page)] = True
        want = 0.5 * was + m
        # products to 2^-20 (see attend64), exponentials and sums of G * n weights to 2^-20, the addition to 2^-24
        limit = bound + m * (2.0 ** -20 + G * max(n, 1) * 2.0 ** -24) + want.abs() * 2.0 ** -23
        assert bool(((got - want).abs() <= limit).all()), (s, float(((got - want).abs() / limit).max()))
    assert bool((out[~seen] == -5.0).all())          # rows that hold no token of the batch


def test_mass_without_prior_and_in_place():
    w = World(2, 128, 96, 4, [150, 90])
    q = queries(w, [1, 5], 4, torch.bfloat16).to(DEV)
    b = w.batch([1, 5], 4)
    once = hqmq.paged_attention_mass(q, w.pool, b, w.tab[0])
    total = torch.stack([torch.cat([once[p] for p in t], 1)[:, :n].sum() for t, n in zip(w.tables, w.kv)]).cpu()
    assert torch.allclose(total, torch.tensor([8.0, 40.0]), atol=1e-3)      # one per query and head
    acc = once.clone()
    hqmq.paged_attention_mass(q, w.pool, b, w.tab[0], prior=acc, out=acc)
    live = torch.zeros_like(once, dtype=torch.bool)
    for t, n in zip(w.tables, w.kv):
        for k, p in enumerate(t):
            live[p, :, :min(64, n - 64 * k)] = True
    assert torch.equal(acc, torch.where(live, once + once, once))


# ---- eviction -----------------------------------------------------------------------------------------------------------------------------
def chosen(mass, n, keep, first, last):
    if keep >= n:
        return list(range(n))
    mid = range(first, n - last)
    heavy = sorted(mid, key=lambda t: (-(mass[t] if mass[t] == mass[t] else -math.inf), math.isnan(mass[t]), t))[:keep - first - last]
    return sorted(list(range(first)) + list(range(n - last, n)) + heavy)


@pytest.mark.parametrize("H,d,S,rb,page,outliers,kv,keep,first,last", [
    (2, 128, 96, 4, 64, "both", [300, 64, 1, 1000], [90, 64, 1, 333], 4, 16),
    (3, 64, 24, 3, 128, "both", [200, 130, 500], [20, 20, 21], 4, 16),
    (1, 128, 192, 6, 64, None, [70, 400], [0, 129], 0, 0),
    (2, 64, 48, 5, 256, "both", [9000, 700], [5000, 255], 1, 0),
    (1, 64, 24, 3, 64, None, [60000], [3000], 0, 7),
])
@pytest.mark.parametrize("kind", ["spread", "ties", "odd"])
def test_eviction(H, d, S, rb, page, outliers, kv, keep, first, last, kind):
    need = sum(-(-n // page) for n in keep)
    w = World(H, d, S, rb, kv, page=page, outliers=outliers, spare=need + 2, rounds=2)
    g = torch.Generator().manual_seed(2)
    mass = torch.rand(w.n_pages, H, page, generator=g) ** 8
    if kind == "ties":
        mass = (mass * 4).round() / 4
    elif kind == "odd":
        u = torch.rand(mass.shape, generator=g)
        mass = mass - 0.5
        for lo, v in ((0.02, float("nan")), (0.04, float("inf")), (0.06, -float("inf")), (0.3, 0.0), (0.5, -0.0)):
            mass = torch.where((u < lo) & (u >= lo - 0.2), torch.tensor(v), mass)
    at, dst = 0, []
    for n in keep:
        dst.append(w.free[at:at + -(-n // page)])
        at += -(-n // page)
    before = [host(w.pool.K), host(w.pool.V)]
    new_mass = torch.full_like(mass, -3.0)
    gm = new_mass.to(DEV)
    src_batch, dst_batch = hqmq.PagedBatch(w.pool, w.tables, kv), hqmq.PagedBatch(w.pool, dst, keep)
    kept = hqmq.paged_evict(w.pool, src_batch, dst_batch, mass.to(DEV), first=first, last=last, out_mass=gm).cpu()
    after, gm = [host(w.pool.K), host(w.pool.V)], gm.cpu()
    assert kept.shape == (len(kv), H, max(keep))
    live = torch.zeros(w.n_pages, page, dtype=torch.bool)
    for s, (n, k) in enumerate(zip(kv, keep)):
        flat = torch.cat([mass[p] for p in w.tables[s]], 1)
        for i in range(k):
            live[dst[s][i // page], i % page] = True
        for h in range(H):
            got = kept[s, h]
            assert got[:k].tolist() == chosen(flat[h].tolist(), n, k, first, last) and bool((got[k:] == -1).all())
            for i, t in enumerate(got[:k].tolist()):
                a, b = (dst[s][i // page], h, i % page), (w.tables[s][t // page], h, t % page)
                for x, y in zip(after, before):
                    assert torch.equal(x["codes"][a], y["codes"][b]) and torch.equal(x["rs"][a], y["rs"][b])
                x, y = gm[a], mass[b]
                assert x == y or (x != x and y != y)
        # the moved tokens decode to what they were, flagged chunks and all
        if n <= 1000:
            for x, y, tab in zip(after, before, w.tab):
                old, new = dense64(y, tab, S, rb, w.tables[s], n), dense64(x, tab, S, rb, dst[s], k) if k else None
                for h in range(H):
                    assert k == 0 or torch.equal(new[h], old[h][kept[s, h, :k].long()])
    # nothing else moved: other pages as they were, rows behind the last token too
    used = torch.zeros(w.n_pages, dtype=torch.bool)
    used[[p for t in dst for p in t]] = True
    for x, y in zip(after, before):
        for name in x:
            if name == "n":
                continue
            u, v = (t.view(torch.int16) if t.dtype in (torch.float16, torch.bfloat16) else t for t in (x[name], y[name]))
            assert torch.equal(u[~used], v[~used]), name
            if name in ("codes", "rs", "flags"):
                m = ~live.view(w.n_pages, 1, page).expand(-1, H, -1)
                assert torch.equal(u[m], v[m]), name
    assert bool((gm.transpose(1, 2)[~live] == -3.0).all())


def test_attention_after_an_eviction_and_an_append():
    w = World(2, 128, 96, 4, [500, 220], spare=12)
    mass = torch.rand(w.n_pages, 2, 64, device=DEV)
    dst = [w.free[:3], w.free[3:6]]
    target = hqmq.PagedBatch(w.pool, dst, [150, 100])
    hqmq.paged_evict(w.pool, w.batch([1, 1], 4), target, mass)
    x = [make_kv("spiky", (1, 2, 3, 128), 77 + i, torch.bfloat16).to(DEV) for i in (0, 1)]
    pair = [w.quant.encode(x[i], 0, i) for i in (0, 1)]
    hqmq.paged_store(w.pool, *pair, hqmq.PagedBatch(w.pool, dst, [152, 101], [2, 1]))
    w.tables, w.kv = dst, [152, 101]
    for q_lens in ([2, 1], [30, 101]):
        q = queries(w, q_lens, 4, torch.bfloat16)
        check_attend(w, hqmq.paged_attention(q.to(DEV), w.pool, w.batch(q_lens, 4), *w.tab), q, q_lens, 4)


# ---- as they are used ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("outliers", [True, False])
def test_paged_cache_agrees_with_the_contiguous_one(outliers):
    """Equal lengths: both caches encode the same tokens with the same medians, so they hold the same codes."""
    B, H, G, d, T = 3, 2, 4, 128, 150
    inner = hqmq.HQMQ(2, H, 96, 4, device=DEV)
    quant = hqmq.with_outlier_extraction(inner, C=3.0) if outliers else inner
    flat = hqmq.PackedKVCache(quant, 400, sliding_window={1: 100})
    paged = hqmq.PagedKVCache(quant, 40, sliding_window={1: 100})
    ids = paged.add(B)
    for step, n in enumerate([T, 1, 1, 20, 1]):
        paged.begin(ids, [n] * B)
        for layer in (0, 1):
            k, v = (make_kv("spiky", (B, H, n, d), 5 * step + layer + 50 * i, torch.bfloat16).to(DEV) for i in (0, 1))
            q = (torch.randn(B, H * G, n, d, generator=torch.Generator().manual_seed(step)) * 1.5).to(torch.bfloat16).to(DEV)
            flat.update(k, v, layer)
            tok = lambda x: x.transpose(1, 2).reshape(B * n, -1, d)
            paged.update(tok(k), tok(v), layer)
            a = flat.attend(q, layer)
            b = paged.attend(tok(q), layer)
            a = tok(a).float()
            assert float((a - b.float()).norm() / a.norm()) < 3 * 2.0 ** -8
    paged.check()
    # the same codes
    pk, pl = flat._layers[0][0], paged.pool(0).K
    rows = pk.codes[:B * H * pk.T_cap * pk.row_bytes].view(B, H, pk.T_cap, -1)
    for s in ids:
        n = paged.length(s)
        got = torch.cat([pl.pages("codes")[p] for p in paged._table[s]], 1)[:, :n]
        assert torch.equal(got, rows[s, :, :n])


def test_paged_cache_serves_sequences_that_come_and_go():
    H, G, d = 2, 4, 64
    quant = hqmq.with_outlier_extraction(hqmq.HQMQ(1, H, 24, 3, device=DEV), C=3.0)
    cache = hqmq.PagedKVCache(quant, 24)
    gen = torch.Generator().manual_seed(0)

    def step(seqs, new):
        cache.begin(seqs, new)
        k, v = (torch.randn(sum(new), H, d, generator=gen).to(torch.bfloat16).to(DEV) for _ in (0, 1))
        cache.update(k, v, 0)
        q = torch.randn(sum(new), H * G, d, generator=gen).to(torch.bfloat16)
        out = cache.attend(q.to(DEV), 0)
        cache.weigh(q.to(DEV), 0, decay=0.9)
        tab = [quant.inner.tables(0, i, DEV)["table16"] for i in (0, 1)]
        K, V = (host(x) for x in (cache.pool(0).K, cache.pool(0).V))
        at = 0
        for s, n in zip(seqs, new):
            if n:
                T = cache.length(s)
                o, _, bound, _ = attend64(q[at:at + n], *(dense64(x, t, 24, 3, cache._table[s], T) for x, t in zip((K, V), tab)), G, None, None, None, d ** -0.5)
                assert bool(((out[at:at + n].cpu().double() - o).abs() <= bound + o.abs() * (2.0 ** -8 + 2.0 ** -18) + 1e-7).all())
            at += n

    a, b, c = cache.add(3)
    step([a, b], [300, 40])
    step([b, c, a], [1, 130, 1])
    step([a, b, c], [1, 0, 1])
    free = cache.free_pages
    kept = cache.evict([a, b, c], keep=100)[0]
    assert kept.shape == (2, H, 100) and [cache.length(s) for s in (a, b, c)] == [100, 41, 100] and cache.free_pages > free
    with pytest.raises(_lib.HqmqError):
        cache.attend(torch.zeros(1, H * G, d, device=DEV), 0)              # the step is over
    step([c, a, b], [30, 1, 2])
    cache.drop([a])
    d_, = cache.add()
    step([d_, b], [60, 1])
    for s in (b, c, d_):
        cache.drop([s])
    assert cache.free_pages == 24
    with pytest.raises(KeyError):
        cache.begin([a], [1])
    e, = cache.add()
    with pytest.raises(_lib.HqmqError):
        cache.begin([e], [24 * 64 + 1])
    assert cache.free_pages == 24 and cache.length(e) == 0


# ---- streams, graphs, refusals ----------------------------------------------------------------------------------------------------------------
def test_another_stream_and_two_calls_at_once():
    w = World(2, 128, 96, 4, [700, 300])
    q = [queries(w, [1, n], 4, torch.bfloat16, seed=n) for n in (1, 40)]
    qd, batches = [x.to(DEV) for x in q], [w.batch([1, n], 4) for n in (1, 40)]
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in q], []
    for _ in range(4):
        for s, x, b in zip(streams, qd, batches):
            with torch.cuda.stream(s):
                outs.append(hqmq.paged_attention(x, w.pool, b, *w.tab))
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        check_attend(w, o, q[i % 2], [1, (1, 40)[i % 2]], 4)


def test_captured_calls_follow_a_renewed_batch():
    kv = [300, 40]
    w = World(2, 128, 96, 4, [1500, 700], garbage=False)
    q = queries(w, [1, 2], 4, torch.bfloat16)
    qd = q.to(DEV)
    b = hqmq.PagedBatch(w.pool, [t[:5] for t in w.tables], kv, [1, 2], n_heads=8, reserve_pages=40)
    out, mass = torch.empty_like(qd), w.pool.new_mass()
    hqmq.paged_attention(qd, w.pool, b, *w.tab, out=out)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        hqmq.paged_attention(qd, w.pool, b, *w.tab, out=out)
        hqmq.paged_attention_mass(qd, w.pool, b, w.tab[0], out=mass)
    full, tables = w.kv, w.tables
    for kv in ([300, 40], [1500, 700], [1, 2], [801, 333]):
        b.renew(tables, kv)
        mass.zero_()
        graph.replay()
        torch.cuda.synchronize()
        w.kv = kv
        w.__dict__.pop("_dense", None)
        check_attend(w, out, q, [1, 2], 4)
        assert abs(float(mass.sum()) - 3 * 8) < 1e-3
    with pytest.raises(ValueError):
        b.renew(tables, [1])


def test_a_batch_is_not_made_inside_a_capture():
    w = World(1, 64, 24, 3, [20], garbage=False)
    graph = torch.cuda.CUDAGraph()
    x = torch.zeros(4, device=DEV)
    with torch.cuda.graph(graph):
        x.add_(1)
        with pytest.raises(_lib.HqmqError):
            w.batch([1], 2)


def test_refusals():
    w = World(2, 128, 96, 4, [100, 50], spare=6)
    b = w.batch([1, 1], 4)
    q = torch.zeros(2, 8, 128, dtype=torch.bfloat16, device=DEV)
    ok = lambda **kw: hqmq.paged_attention(kw.pop("Q", q), w.pool, kw.pop("batch", b), *kw.pop("tab", w.tab), **kw)
    ok()
    other = World(2, 128, 24, 3, [100, 50])
    for kw in (dict(Q=q[:1]), dict(Q=q[:, :4]), dict(Q=q[..., :64]), dict(batch=other.batch([1, 1], 4)), dict(tab=other.tab),
               dict(tab=[t.float() for t in w.tab]), dict(softcap=0.0), dict(softcap=-3.0), dict(softcap=float("nan")),
               dict(sinks=torch.zeros(4, device=DEV)), dict(out=torch.empty(2, 8, 64, device=DEV)),
               dict(batch=hqmq.PagedBatch(w.pool, w.tables, w.kv))):
        with pytest.raises(ValueError):
            ok(**kw)
    with pytest.raises(_lib.HqmqError):
        ok(out=torch.empty(2, 8, 256, device=DEV)[..., ::2])
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            ok(softmax_scale=scale)
    with pytest.raises(TypeError):
        ok(Q=q.to(torch.int32))
    with pytest.raises(TypeError):
        hqmq.paged_attention_mass(q.float(), w.pool, b, w.tab[0])
    for kw in (dict(prior=torch.zeros(3, device=DEV)), dict(out=w.pool.new_mass().double()), dict(decay=float("inf"))):
        with pytest.raises(ValueError):
            hqmq.paged_attention_mass(q, w.pool, b, w.tab[0], **kw)
    mass, f = w.pool.new_mass(), w.free
    src = hqmq.PagedBatch(w.pool, w.tables, w.kv)
    evict = lambda tables, kv, **kw: hqmq.paged_evict(w.pool, src, hqmq.PagedBatch(w.pool, tables, kv), mass, **kw)
    for tables, kv, kw in (([f[:2], f[2:3]], [101, 50], {}), ([f[:1], f[1:2]], [19, 50], {}), ([f[:1], f[:1]], [30, 30], {}),
                           ([w.tables[0][:1], f[:1]], [30, 30], {}), ([f[:1]], [30], {}), ([f[:1], f[1:2]], [30, 30], dict(first=-1)),
                           ([f[:1], f[1:2]], [30, 30], dict(out_mass=mass[:1]))):
        with pytest.raises(ValueError):
            evict(tables, kv, **kw)
    pair = [w.quant.encode(torch.randn(1, 2, 2, 128, device=DEV).to(torch.bfloat16), 0, i) for i in (0, 1)]
    with pytest.raises(ValueError):
        hqmq.paged_store(w.pool, *pair, hqmq.PagedBatch(w.pool, w.tables, w.kv, [2, 1]))            # three tokens
    with pytest.raises(ValueError):
        hqmq.paged_store(w.pool, *pair, hqmq.PagedBatch(w.pool, [f[:2], f[:2]], [80, 80], [1, 1]))   # into one page
    half = [w.quant.encode(torch.randn(1, 2, 2, 128, device=DEV).half(), 0, i) for i in (0, 1)]
    with pytest.raises(ValueError):
        hqmq.paged_store(w.pool, *half, hqmq.PagedBatch(w.pool, w.tables, w.kv, [1, 1]))


def test_nothing_to_do():
    w = World(1, 64, 24, 3, [100, 30], spare=3)
    b = hqmq.PagedBatch(w.pool, w.tables, w.kv, [0, 0], n_heads=2)
    q = torch.zeros(0, 2, 64, dtype=torch.bfloat16, device=DEV)
    assert hqmq.paged_attention(q, w.pool, b, *w.tab).shape == (0, 2, 64)
    mass = hqmq.paged_attention_mass(q, w.pool, b, w.tab[0], prior=torch.ones_like(w.pool.new_mass()), decay=0.5)
    assert float(mass.sum()) == 0.5 * 130
    empty = hqmq.PagedBatch(w.pool, [[], []], [0, 0])
    assert hqmq.paged_evict(w.pool, hqmq.PagedBatch(w.pool, w.tables, w.kv), empty, mass, first=0, last=0).shape == (2, 1, 0)


# ---- tokens that are stored again -------------------------------------------------------------------------------------------------------------
def _same_contents(a, b, tables, kv):
    """Two pools hold the same tokens: rows, scales, flags, offsets, counts and the entries that those reach."""
    page = a.page_tokens
    for x, y in zip((host(a.K), host(a.V)), (host(b.K), host(b.V))):
        for t, n in zip(tables, kv):
            for k, p in enumerate(t[:-(-n // page)]):
                m = min(page, n - k * page)
                for name in ("codes", "rs", "flags"):
                    assert torch.equal(x[name][p, :, :m], y[name][p, :, :m]), name
                assert torch.equal(x["out_count"][p], y["out_count"][p])
                assert torch.equal(x["out_off"][p, :, :-(-m // 16) + 1], y["out_off"][p, :, :-(-m // 16) + 1])
                for h in range(x["codes"].shape[1]):
                    e = int(x["out_count"][p, h])
                    assert torch.equal(x["out_vals"][p, h, :e], y["out_vals"][p, h, :e])


@pytest.mark.parametrize("H,d,S,rb,page", [(2, 128, 96, 4, 64), (1, 64, 24, 3, 128)])
@pytest.mark.parametrize("length,drafted,taken", [(96, 4, 2), (92, 4, 4), (94, 4, 2), (62, 4, 3), (60, 70, 66), (127, 1, 1), (64, 3, 3), (20, 4, 3)])
def test_tokens_that_were_taken_back_leave_nothing(H, d, S, rb, page, length, drafted, taken):
    """`drafted` tokens behind `length`, of which the last `taken` are rejected; others follow: a pool that never held them holds the same."""
    q = hqmq.HQMQ(1, H, S, rb, device=DEV)
    quant = hqmq.with_outlier_extraction(q, C=1.5)
    pools = [hqmq.PagedKV(8, H, d, S, rb, DEV, page_tokens=page, outliers_K=True, outliers_V=True, out_cap=page * d // 4) for _ in (0, 1)]
    tables = [[5, 2, 7, 1][:-(-(length + 4 + drafted) // page)], [0]]

    def encoded(n, seed):
        x = [make_kv("spiky", (1, H, n, d), seed + i, torch.bfloat16).to(DEV) for i in (0, 1)]
        pair = [q.new_cache(1, n, d, DEV, scale_dtype=torch.bfloat16, with_outliers=True, out_dtype=torch.bfloat16) for _ in (0, 1)]
        quant.encode_pair(*x, 0, *pair)
        return pair

    def store(pool, pair, kv, new):
        hqmq.paged_store(pool, *pair, hqmq.PagedBatch(pool, tables, kv, new))

    keep = drafted - taken
    first, draft, other, more = encoded(length + 40, 1), encoded(drafted, 3), encoded(1, 5), encoded(3, 7)
    for i, pool in enumerate(pools):
        store(pool, first, [length, 40], [length, 40])
        if i == 0:
            for _ in (0, 1):                     # (the same step twice)
                store(pool, draft, [length + drafted, 40], [drafted, 0])
                store(pool, other, [length + drafted, 41], [0, 1])
        else:
            if keep:
                store(pool, draft, [length + keep, 40], [keep, 0])
            store(pool, other, [length + keep, 41], [0, 1])
        store(pool, more, [length + keep + 2, 42], [2, 1])
    kv = [length + keep + 2, 42]
    _same_contents(*pools, tables, kv)
    Q = torch.randn(2, 4 * H, d, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(DEV)
    tab = [q.tables(0, i, DEV)["table16"] for i in (0, 1)]
    a, b = (hqmq.paged_attention(Q, p, hqmq.PagedBatch(p, tables, kv, [1, 1], n_heads=4 * H), *tab) for p in pools)
    assert torch.equal(a, b)


@pytest.mark.parametrize("power", [16, 24, 32, 40, 90])
@pytest.mark.parametrize("q_lens", [[1, 1], [60, 33]])
def test_scores_that_no_exponential_holds(power, q_lens):
    """Scores up to 2^95: the largest one takes the weight."""
    w = World(1, 128, 96, 4, [200, 90])
    q = (queries(w, q_lens, 4, torch.bfloat16).float() * 2.0 ** power).to(torch.bfloat16)
    out = hqmq.paged_attention(q.to(DEV), w.pool, w.batch(q_lens, 4), *w.tab)
    assert bool(out.isfinite().all())
    check_attend(w, out, q, q_lens, 4)
    # a key that is far ahead of the others: its value, alone
    K, V = w.dense()
    at = 0
    for s, n in enumerate(q_lens):
        score = torch.einsum("ihd,td->iht", q[at:at + n].double(), K[s][0])
        score = score.masked_fill(torch.arange(w.kv[s]) > torch.arange(n).view(-1, 1, 1) + w.kv[s] - n, -math.inf)
        size = torch.einsum("ihd,td->iht", q[at:at + n].double().abs(), K[s][0].abs()).amax(-1)
        top = score.topk(2, -1)
        sure = (top.values[..., 0] - top.values[..., 1] > size * 2.0 ** -9) & (top.values[..., 1] > -math.inf)
        want = V[s][0][top.indices[..., 0]]
        off = (out[at:at + n].cpu().double() - want).abs()
        assert bool(sure.any()) and bool((off <= want.abs() * (2.0 ** -8 + 2.0 ** -9) + V[s].abs().amax() * 2.0 ** -24)[sure].all())
        at += n


# ---- rows that have nothing to do with one another ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("d,q_dtype", [(128, torch.bfloat16), (64, torch.bfloat16), (128, torch.float32)])
@pytest.mark.parametrize("q_lens", [[1, 1], [4, 8], [60, 33]])
def test_queries_of_sizes_far_from_one_another(d, q_dtype, q_lens):
    """Rows from 2^-40 to 2^110 side by side: every one has the bits that it would have alone."""
    w = World(1, d, 96, 4, [200, 90])
    q = queries(w, q_lens, 4, torch.bfloat16)
    powers = torch.tensor([0, 20, -40, 3, 60, 0, 110, -1, 12])[torch.arange(4 * sum(q_lens)) % 9].view(-1, 4, 1)
    q = (q.double() * 2.0 ** powers.double()).to(q_dtype)
    view = torch.zeros(sum(q_lens), 4, d + 1, dtype=q_dtype)
    view[..., 1:] = q
    for x in (q.to(DEV), view.to(DEV)[..., 1:]):             # (wide loads, and an element at a time)
        check_attend(w, hqmq.paged_attention(x, w.pool, w.batch(q_lens, 4), *w.tab), q, q_lens, 4)


@pytest.mark.parametrize("q_dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("q_lens", [[1, 1], [4, 8], [60, 33]])
def test_queries_that_are_no_numbers_spoil_their_own_rows_only(q_dtype, q_lens):
    w = World(2, 128, 96, 4, [200, 90])
    q = queries(w, q_lens, 4, q_dtype)
    bad = torch.zeros(q.shape[:2], dtype=torch.bool)
    for i, (row, head, value) in enumerate(((0, 1, math.inf), (-1, 6, -math.inf), (sum(q_lens) // 2, 4, math.nan))):
        q[row, head, 5 + 30 * i] = value
        bad[row, head] = True
    out = hqmq.paged_attention(q.to(DEV), w.pool, w.batch(q_lens, 4), *w.tab).cpu()
    K, V = w.dense()
    at = 0
    for s, n in enumerate(q_lens):
        clean = torch.where(bad[at:at + n, :, None], torch.zeros((), dtype=q_dtype), q[at:at + n])
        o, _, bound, _ = attend64(clean, K[s], V[s], 4, None, None, None, 128 ** -0.5)
        off = (out[at:at + n].double() - o).abs()
        fine = off <= bound + o.abs() * (HALF[q_dtype] + 2.0 ** -18) + 1e-7
        assert bool(fine[~bad[at:at + n]].all())
        assert bool(out[at:at + n][bad[at:at + n]].isnan().all())
        at += n


def test_a_prompt_whose_weights_have_no_room():
    n, G, d = 190_000, 16, 64
    w = World(1, d, 24, 3, [n], outliers=None, rounds=1, page=1024, kind="randn", garbage=False)
    b = w.batch([n], G)
    q = (1.5 * torch.randn(n, G, d, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))).to(torch.bfloat16)
    out = hqmq.paged_attention(q, w.pool, b, *w.tab)
    with pytest.raises(ValueError, match="no room"):
        hqmq.paged_attention_mass(q, w.pool, b, w.tab[0])
    (K,), (V,) = w.dense()
    for t in (0, 31, 5000, 100_001, n - 1):
        o, _, bound, _ = attend64(q[t:t + 1].cpu(), K[:, :t + 1], V[:, :t + 1], G, None, None, None, d ** -0.5)
        assert bool(((out[t:t + 1].cpu().double() - o).abs() <= bound + o.abs() * (2.0 ** -8 + 2.0 ** -18) + 1e-7).all()), t


def test_a_decay_that_fp32_does_not_hold_is_refused():
    w = World(1, 64, 24, 3, [40], garbage=False)
    q = torch.zeros(1, 2, 64, dtype=torch.bfloat16, device=DEV)
    for decay in (1e300, -1e39, float("nan")):
        with pytest.raises(ValueError):
            hqmq.paged_attention_mass(q, w.pool, w.batch([1], 2), w.tab[0], decay=decay)


def test_a_cache_of_layers_with_different_head_dims():
    H, G, dims = 2, 4, (128, 64)
    inner = hqmq.HQMQ(2, H, 24, 3, device=DEV)
    cache = hqmq.PagedKVCache(inner, 24)
    ids, gen = cache.add(2), torch.Generator().manual_seed(0)
    for new in ([300, 40], [1, 2]):
        cache.begin(ids, new)
        for layer, d in enumerate(dims):
            k, v = (torch.randn(sum(new), H, d, generator=gen).to(torch.bfloat16).to(DEV) for _ in (0, 1))
            cache.update(k, v, layer)
            q = torch.randn(sum(new), H * G, d, generator=gen).to(torch.bfloat16)
            out = cache.attend(q.to(DEV), layer).cpu()
            cache.weigh(q.to(DEV), layer)
            tabs = [inner.tables(layer, i, DEV)["table16"] for i in (0, 1)]
            at = 0
            for s, n in zip(ids, new):
                K, V = (dense64(host(x), t, 24, 3, cache._table[s], cache.length(s)) for x, t in zip((cache.pool(layer).K, cache.pool(layer).V), tabs))
                o, _, bound, _ = attend64(q[at:at + n], K, V, G, None, None, None, d ** -0.5)
                assert bool(((out[at:at + n].double() - o).abs() <= bound + o.abs() * (2.0 ** -8 + 2.0 ** -18) + 1e-7).all())
                at += n
    kept = cache.evict(ids, keep=100)
    assert sorted(kept) == [0, 1] and all(k.shape == (1, H, 100) for k in kept.values()) and [cache.length(s) for s in ids] == [100, 42]


@pytest.mark.parametrize("kind", ["spread", "ties"])
def test_eviction_of_a_sequence_longer_than_shared_memory_holds(kind):
    """More than eight CTAs' weights (327680), beside short sequences of the same call."""
    kv, keep, first, last, page = [340_001, 700, 12_345], [20_000, 100, 12_345], 4, 16, 1024
    need = [-(-n // page) for n in kv + keep]
    order = list(range(sum(need)))
    random.Random(0).shuffle(order)
    cuts = np.cumsum([0] + need)
    tables = [order[a:z] for a, z in zip(cuts, cuts[1:])]
    pool = hqmq.PagedKV(sum(need), 1, 64, 24, 3, DEV, page_tokens=page)
    g = torch.Generator(device=DEV).manual_seed(1)
    for pk in (pool.K, pool.V):
        pk.pages("codes").random_(0, 256, generator=g)
        pk.pages("rs").uniform_(generator=g)
    mass = torch.rand(sum(need), 1, page, device=DEV, generator=g)
    if kind == "ties":
        mass = (mass * 4).round()
    before = [{k: v.cpu() for k, v in pk.planes().items()} for pk in (pool.K, pool.V)]
    was = mass.cpu()
    kept = hqmq.paged_evict(pool, hqmq.PagedBatch(pool, tables[:3], kv), hqmq.PagedBatch(pool, tables[3:], keep), mass, first=first, last=last).cpu()
    now = mass.cpu()
    for s, (n, k) in enumerate(zip(kv, keep)):
        flat = torch.cat([was[p, 0] for p in tables[s]])[:n].double().numpy()
        mid = np.argsort(-flat[first:n - last], kind="stable")[:k - first - last] + first
        want = np.sort(np.concatenate([np.arange(first), mid, np.arange(n - last, n)])) if k < n else np.arange(n)
        assert kept[s, 0, :k].tolist() == want.tolist() and bool((kept[s, 0, k:] == -1).all())
        src = torch.tensor(tables[s])[torch.from_numpy(want) // page], torch.from_numpy(want) % page
        dst = torch.tensor(tables[3 + s])[torch.arange(k) // page], torch.arange(k) % page
        for x, y in zip((pool.K, pool.V), before):
            for name in ("codes", "rs"):
                assert torch.equal(x.pages(name).cpu()[dst[0], 0, dst[1]], y[name][src[0], 0, src[1]])
        assert torch.equal(now[dst[0], 0, dst[1]], was[src[0], 0, src[1]])


@pytest.mark.parametrize("value", [math.inf, math.nan])
@pytest.mark.parametrize("q_lens,token", [([1, 8], 85), ([33, 60], 50), ([150, 90], 2)])
def test_a_key_that_is_no_number_spoils_the_queries_that_see_it_only(value, q_lens, token):
    w = World(1, 128, 96, 4, [200, 90])
    K, V = w.dense()
    w.pool.K.pages("rs")[w.tables[1][token // 64], 0, token % 64] = value
    q = queries(w, q_lens, 4, torch.bfloat16)
    out = hqmq.paged_attention(q.to(DEV), w.pool, w.batch(q_lens, 4), *w.tab).cpu()
    at = 0
    for s, n in enumerate(q_lens):
        o, _, bound, _ = attend64(q[at:at + n], K[s], V[s], 4, None, None, None, 128 ** -0.5)
        fine = (out[at:at + n].double() - o).abs() <= bound + o.abs() * (2.0 ** -8 + 2.0 ** -18) + 1e-7
        first = max(0, token - (w.kv[s] - n)) if s else n                        # the first query that sees the key
        assert bool(fine[:first].all()) and bool(out[at + first:at + n].isnan().all()), s
        at += n


@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_weights_beside_a_key_that_is_no_number(value):
    """A sequence whose queries see it has no weights; the other one has its own."""
    w = World(1, 128, 96, 4, [200, 90])
    K, V = w.dense()
    w.pool.K.pages("rs")[w.tables[1][0], 0, 30] = value
    for q_lens in ([1, 1], [12, 3]):
        q = queries(w, q_lens, 4, torch.bfloat16)
        mass = hqmq.paged_attention_mass(q.to(DEV), w.pool, w.batch(q_lens, 4), w.tab[0]).cpu()
        _, m, _, bound = attend64(q[:q_lens[0]], K[0], V[0], 4, None, None, None, 128 ** -0.5)
        got = [torch.cat([mass[p] for p in t], 1)[:, :n].double() for t, n in zip(w.tables, w.kv)]
        assert bool(((got[0] - m).abs() <= bound + m * (2.0 ** -20 + 4 * q_lens[0] * 2.0 ** -24)).all())
        assert bool(got[1].isnan().all())


@pytest.mark.parametrize("d,S,rb", [(128, 96, 4), (64, 96, 4), (128, 192, 6)])
@pytest.mark.parametrize("channels", [1, 2, 3, 4, 5])
def test_chunk_columns_that_most_tokens_have_flagged(d, S, rb, channels):
    """About 13 to 70 flagged chunks a tile, in K and V: as many as a warp has table entries for, as are staged, and more."""
    w = World(1, d, S, rb, [300, 90, 17], rounds=1, kind="randn", garbage=False)
    x = [make_kv("randn", (1, 1, 407, d), 5 + i, torch.bfloat16) for i in (0, 1)]
    for y in x:
        y[..., torch.arange(channels) * 8 + 3] *= 40.0
    pair = [w.quant.encode(y.to(DEV), 0, i) for i, y in enumerate(x)]
    hqmq.paged_store(w.pool, *pair, hqmq.PagedBatch(w.pool, w.tables, w.kv, w.kv))
    for q_lens in ([1, 1, 1], [4, 3, 1], [8, 2, 1]):
        q = queries(w, q_lens, 4, torch.bfloat16)
        check_attend(w, hqmq.paged_attention(q.to(DEV), w.pool, w.batch(q_lens, 4), *w.tab), q, q_lens, 4)


def test_captured_steps_store_and_attend():
    """A step captured once and replayed: its tokens are stored where the renewed batch says, whatever warm-up calls stored before."""
    H, G, d, B = 2, 4, 128, 2
    q = hqmq.HQMQ(1, H, 96, 4, device=DEV)
    quant = hqmq.with_outlier_extraction(q, C=1.5)
    tab = [q.tables(0, i, DEV)["table16"] for i in (0, 1)]
    pools = [hqmq.PagedKV(12, H, d, 96, 4, DEV, outliers_K=True, outliers_V=True, out_cap=64 * 32) for _ in (0, 1)]
    tables, kv, n_new = [[3, 1, 7], [0, 5, 9]], [61, 20], [1, 2]
    x = [make_kv("spiky", (1, H, sum(kv), d), i, torch.bfloat16).to(DEV) for i in (0, 1)]
    first = [q.new_cache(1, sum(kv), d, DEV, scale_dtype=torch.bfloat16, with_outliers=True, out_dtype=torch.bfloat16) for _ in (0, 1)]
    quant.encode_pair(*x, 0, *first)
    for pool in pools:
        hqmq.paged_store(pool, *first, hqmq.PagedBatch(pool, tables, kv, kv))
    pair = [q.new_cache(1, sum(n_new), d, DEV, scale_dtype=torch.bfloat16, with_outliers=True, out_dtype=torch.bfloat16) for _ in (0, 1)]
    fresh = lambda seed: [make_kv("spiky", (1, H, sum(n_new), d), seed + i, torch.bfloat16).to(DEV) for i in (0, 1)]
    quant.encode_pair(*fresh(50), 0, *pair)
    Q = torch.randn(sum(n_new), H * G, d, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(DEV)
    batch = hqmq.PagedBatch(pools[0], tables, [n + m for n, m in zip(kv, n_new)], n_new, n_heads=H * G, reserve_pages=12)
    out = torch.empty_like(Q)

    def step():
        hqmq.paged_store(pools[0], *pair, batch)
        hqmq.paged_attention(Q, pools[0], batch, *tab, out=out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(6):                                                   # (over the end of a page and of blocks)
        kv = [n + m for n, m in zip(kv, n_new)]
        new = [q.new_cache(1, sum(n_new), d, DEV, scale_dtype=torch.bfloat16, with_outliers=True, out_dtype=torch.bfloat16) for _ in (0, 1)]
        quant.encode_pair(*fresh(60 + 2 * i), 0, *new)
        for a, b in zip(pair, new):
            for name in ("codes", "rs", "flags", "out_off", "out_vals"):
                getattr(a, name).copy_(getattr(b, name))
        batch.renew(tables, kv)
        graph.replay()
        eager = hqmq.PagedBatch(pools[1], tables, kv, n_new, n_heads=H * G)
        hqmq.paged_store(pools[1], *new, eager)
        want = hqmq.paged_attention(Q, pools[1], eager, *tab)
        torch.cuda.synchronize()
        _same_contents(*pools, tables, kv)
        assert float((out.float() - want.float()).abs().max()) <= 2.0 ** -7 * float(want.float().abs().max())
