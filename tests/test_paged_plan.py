"""Plans of calls over a paged cache (host code), their refusals, and those of the calls, without a GPU."""
import ctypes as C
import os
import random
import re

import numpy as np
import pytest
import torch

import hqmq_b200 as hqmq
from hqmq_b200 import _lib

DEC_WARPS, DEC_WARPS_WIDE, MASS_WARPS = 16, 8, 12


def make_pool(n_pages=64, H=2, d=128, S=24, rb=3, page=64, **kw):
    return hqmq.PagedKV(n_pages, H, d, S, rb, "cpu", page_tokens=page, **kw)


def tables_for(kv, page, n_pages, rng):
    order = list(range(n_pages))
    rng.shuffle(order)
    out, at = [], 0
    for n in kv:
        k = -(-n // page)
        out.append(order[at:at + k])
        at += k
    return out


def keys_of(kv, q, G, window, row0, row1):
    first, last = kv - q + row0 // G, kv - q + (row1 - 1) // G
    return (max(0, first + 1 - window) if window else 0), last + 1


def stretch(w, total, n):
    n = min(n, total)
    return w * total // n if w < n else total


def check_flat(words, units, bases, warps, total, ctas, per_cta, want, tables, page, lengths):
    """Units in order with their tile ranges, prefix sums, and the unit that every warp's stretch begins in."""
    got = [tuple(words[units + 4 * i:units + 4 * i + 4].tolist()) for i in range(len(want))]
    assert got == want
    base = np.cumsum([0] + [u[3] - u[2] for u in want])
    assert words[bases:bases + len(want) + 1].tolist() == base.tolist() and base[-1] == total
    n = ctas * per_cta
    for w in range(n):
        f = stretch(w, total, n)
        rec = words[warps + 16 * w:warps + 16 * w + 16].tolist()
        assert rec[:2] == [f, stretch(w + 1, total, n)]
        if f < total:
            u = rec[2]
            assert base[u] <= f < base[u + 1] and rec[3:5] == [want[u][2] + f - base[u], want[u][3]]
            s = want[u][0]
            tab = sum(len(t) for t in tables[:s])
            assert rec[5:8] == [tab, tables[s][rec[3] * 16 // page], want[u][1]] and rec[8:10] == base[u:u + 2].tolist()
            assert rec[12:14] == lengths[s] and rec[15] == tab


@pytest.mark.parametrize("seed", range(12))
def test_plan_covers_every_tile_once(seed):
    rng = random.Random(seed)
    H, G, d = rng.choice([(1, 1, 64), (2, 4, 128), (4, 7, 128), (8, 8, 64), (3, 16, 64)])
    page, window = rng.choice([64, 128, 256]), rng.choice([0, 1, 100, 128])
    B = rng.randint(1, 9)
    kv = [rng.choice([0, 1, rng.randint(1, 40), rng.randint(1, 900)]) for _ in range(B)]
    q = [min(n, rng.choice([0, 1, 1, 2, 5, 130, 400])) for n in kv]
    n_pages = sum(-(-n // page) for n in kv) + 2
    pool = make_pool(n_pages, H, d, page=page)
    tables = tables_for(kv, page, n_pages, rng)
    b = hqmq.PagedBatch(pool, tables, kv, q, n_heads=H * G, window=window or None)
    p, w = b.plan, b.data.numpy()
    assert p.total_q == sum(q) and len(w) == p.words
    # sequences and tables
    at = 0
    for s in range(B):
        n, nq, off, tab = w[p.seqs + 4 * s:p.seqs + 4 * s + 4]
        assert (n, nq, off) == (kv[s], q[s], at)
        assert w[p.tabs + tab:p.tabs + tab + len(tables[s])].tolist() == tables[s]
        at += q[s]
    tiles = lambda lo, hi: (lo // 16, -(-hi // 16))
    few = [s for s in range(B) if 0 < q[s] * G <= 32]
    dec = [(s, 0, *tiles(*keys_of(kv[s], q[s], G, window, 0, q[s] * G))) for s in few]
    assert p.dec_units == len(dec) and p.dec_rows == next(r for r in (8, 16, 32) if all(q[s] * G <= r for s in few))
    if dec:
        per = DEC_WARPS_WIDE if p.dec_rows > 8 else DEC_WARPS
        check_flat(w, p.dec_unit, p.dec_base, p.dec_warp, p.dec_tiles, p.dec_ctas, per, dec, tables, page, [list(x) for x in zip(kv, q)])
        # units between CTAs: every cut names its first and last CTA
        base = w[p.dec_base:p.dec_base + len(dec) + 1]
        n = p.dec_ctas * per
        edges = [stretch(c * per, p.dec_tiles, n) for c in range(p.dec_ctas + 1)]
        cta = lambda f: max(c for c in range(p.dec_ctas) if edges[c] <= f and edges[c] < edges[c + 1])
        cuts = [(u, cta(base[u]), cta(base[u + 1] - 1)) for u in range(len(dec))]
        want = [(u, a, z, int(base[u] > edges[a])) for u, a, z in cuts if a != z]
        assert [tuple(w[p.dec_cut + 4 * i:p.dec_cut + 4 * i + 4].tolist()) for i in range(w[5])] == want
    # attention weights: row blocks of every sequence, groups of tokens
    rows = p.ms_rows
    ms = [(s, r, *tiles(*keys_of(kv[s], q[s], G, window, r, min(q[s] * G, r + rows)))) for s in range(B) for r in range(0, q[s] * G, rows)]
    assert p.ms_units == len(ms)
    if ms:
        check_flat(w, p.ms_unit, p.ms_base, p.ms_warp, p.ms_tiles, p.ms_ctas, MASS_WARPS, ms, tables, page, [list(x) for x in zip(kv, q)])
    groups = [w[p.ms_group + 4 * i:p.ms_group + 4 * i + 4].tolist() for i in range(p.ms_groups)]
    assert [g[:2] for g in groups] == [[s, t] for s in range(B) for t in range(0, kv[s], 512 if rows == 8 else 128)]
    for s, t, u0, u1 in groups:
        assert [u for u in range(len(ms)) if ms[u][0] == s] == list(range(u0, u1))
    # prompt chunks: units of a sequence in order, images of the tiles that any of them sees, pieces of equal size
    P, units = 128 // G, []
    chunks = [s for s in range(B) if q[s] * G > 32]
    per = p.ch_streams * P
    img = 0
    for i, s in enumerate(chunks):
        mine = []
        for m in range(-(-q[s] // per)):
            lo, hi = keys_of(kv[s], q[s], 1, window, m * per, min(q[s], (m + 1) * per))
            mine.append((s, m, lo // 128, max(1, -(-hi // 128) - lo // 128)))
        first, last = min(u[2] for u in mine), max(u[2] + u[3] for u in mine)
        assert w[p.ch_img + 4 * i:p.ch_img + 4 * i + 4].tolist() == [s, first, last - first, img]
        off = sum(q[:s])
        units += [[*u, kv[s], q[s], off, img - first] for u in mine]
        img += last - first
    assert [w[p.ch_unit + 8 * i:p.ch_unit + 8 * i + 8].tolist() for i in range(p.ch_units)] == units
    assert p.ch_img_tiles == img and p.ch_tiles == sum(u[3] for u in units) and (not units or p.H_kv % p.ch_heads == 0)
    if units and p.ch_whole:
        order = w[p.ch_order:p.ch_order + len(units)].tolist()
        assert sorted(order) == list(range(len(units))) and all(units[a][3] >= units[z][3] for a, z in zip(order, order[1:]))
    elif units:
        flat = [(h, m, o) for h in range(p.ch_heads) for m in range(len(units)) for o in range(units[m][3])]
        L = -(-len(flat) // p.ch_ctas)
        assert [tuple(w[p.ch_start + 4 * c:p.ch_start + 4 * c + 3].tolist()) for c in range(p.ch_ctas)] == [flat[c * L] for c in range(p.ch_ctas)]


@pytest.mark.parametrize("kv,q,kw", [
    ([10], [11], {}),                                # more new tokens than tokens
    ([-1], [0], {}),
    ([10, 10], [1], {}),
    ([10], [1], dict(window=0)),
    ([10], [1], dict(n_heads=3)),
    ([65], [1], {}),                                 # one page named, two needed
])
def test_batches_that_are_refused(kv, q, kw):
    pool = make_pool()
    with pytest.raises(ValueError):
        hqmq.PagedBatch(pool, [[0]] * len(kv), kv, q, **{"n_heads": 4, **kw})


@pytest.mark.parametrize("page", [-1, 64, 1 << 20])
def test_pages_outside_of_the_pool_are_refused(page):
    pool = make_pool(64)
    with pytest.raises(ValueError):
        hqmq.PagedBatch(pool, [[0, page]], [100], [1], n_heads=4)
    hqmq.PagedBatch(pool, [[0, page]], [64], [1], n_heads=4)        # (an entry behind the last page is not read)
    plan = _lib.PagedPlan(struct_size=C.sizeof(_lib.PagedPlan), n_seqs=1, n_pages=64, page_tokens=64, H_q=4, H_kv=2, d=128)
    kv, q, tab = (np.array(x, dtype=np.int32) for x in ([100], [1], [0, page]))
    L = _lib.lib()
    assert L.hqmq_paged_plan_size(C.byref(plan), kv.ctypes.data, q.ctypes.data) == 0
    out = np.zeros(plan.words, dtype=np.int32)
    assert L.hqmq_paged_plan_fill(C.byref(plan), kv.ctypes.data, q.ctypes.data, tab.ctypes.data, 2, out.ctypes.data) == -2


def test_more_refusals_of_batches():
    pool = make_pool()
    with pytest.raises(TypeError):
        hqmq.PagedBatch(pool, [[0]], [1.5], [1], n_heads=4)
    with pytest.raises(ValueError):
        hqmq.PagedBatch(pool, [[0]], [1 << 40], [1], n_heads=4)
    with pytest.raises(ValueError):
        hqmq.PagedBatch(pool, [], [], [])
    with pytest.raises(_lib.HqmqError):
        hqmq.PagedBatch(pool, [[0, 1]], [100], [1], n_heads=4, reserve_pages=1)
    with pytest.raises(_lib.HqmqError):
        hqmq.PagedBatch(pool, [[0]], [10], [1], n_heads=2 * 17)       # 17 query heads per KV head
    with pytest.raises(_lib.HqmqError):
        hqmq.PagedBatch(pool, [[0]], [10], [1], n_heads=4).renew([[0]], [11])
    for bad in (dict(page_tokens=96), dict(page_tokens=2048), dict(dtype=torch.float32)):
        with pytest.raises((ValueError, TypeError)):
            hqmq.PagedKV(4, 2, 128, 24, 3, "cpu", **bad)
    with pytest.raises(ValueError):
        hqmq.PagedKV(4, 2, 96, 24, 3, "cpu")


def test_tables_in_any_form():
    pool = make_pool()
    want = hqmq.PagedBatch(pool, [[5, 3], [7]], [100, 9], n_heads=4).data
    for t in (np.array([[5, 3], [7, 99]]), torch.tensor([[5, 3, -1], [7, -1, -1]]), ((5, 3, 8), (7,)), [torch.tensor([5, 3]), torch.tensor([7, 0])]):
        assert torch.equal(hqmq.PagedBatch(pool, t, torch.tensor([100, 9]), n_heads=4).data, want)


def test_a_plan_with_room_keeps_its_places():
    pool = make_pool(200, H=2)
    rng = random.Random(3)
    b = hqmq.PagedBatch(pool, tables_for([300, 40], 64, 200, rng), [300, 40], [1, 2], n_heads=8, window=None, reserve_pages=60)
    before = {n: getattr(b.plan, n) for n, _ in _lib.PagedPlan._fields_}
    p = _lib.PagedPlan.from_buffer_copy(b.plan)
    p.renew = 1
    same = set(before) - {"n_tab", "dec_tiles", "ms_tiles", "ms_groups", "renew"}
    for kv in ([301, 41], [3000, 700], [1, 2]):
        t = tables_for(kv, 64, 200, rng)
        host, *_ = b._lay_out(p, t, kv, [1, 2])
        assert all(getattr(p, n) == before[n] for n in same)
        w = host.numpy()
        assert w[1] == p.dec_tiles == sum(-(-n // 16) for n in kv) and w[p.tabs:p.tabs + len(t[0])].tolist() == t[0]
    with pytest.raises(_lib.HqmqError):
        b._lay_out(p, tables_for([3000, 900], 64, 200, rng), [3000, 900], [1, 2])       # 62 pages
    with pytest.raises(_lib.HqmqError):
        b._lay_out(p, [[0], [1]], [20, 20], [1, 1])
    c = hqmq.PagedBatch(pool, [[1, 2]], [100], [50], n_heads=8, reserve_pages=10)       # a prompt chunk
    p = _lib.PagedPlan.from_buffer_copy(c.plan)
    p.renew = 1
    with pytest.raises(_lib.HqmqError):
        c._lay_out(p, [[1, 2]], [101], [50])


def test_pages_shared_and_written():
    pool = make_pool()
    shared = hqmq.PagedBatch(pool, [[1, 2], [1, 3]], [100, 90], [1, 1])      # a common prefix; new tokens in pages of their own
    assert shared.stores_alone() and not shared._unshared
    assert not hqmq.PagedBatch(pool, [[1, 2], [1, 2]], [100, 90], [1, 1]).stores_alone()
    assert not hqmq.PagedBatch(pool, [[1, 1]], [100], [1]).stores_alone()
    assert hqmq.PagedBatch(pool, [[1, 2], [2]], [100, 0], [1, 0]).stores_alone()


def test_calls_refuse_host_memory():
    pool = make_pool()
    b = hqmq.PagedBatch(pool, [[0]], [10], [1], n_heads=4)
    t = torch.zeros(2, 24 * 24, 4, dtype=torch.float16)
    for call in (lambda: hqmq.paged_attention(torch.zeros(1, 4, 128), pool, b, t, t),
                 lambda: hqmq.paged_attention_mass(torch.zeros(1, 4, 128), pool, b, t),
                 lambda: hqmq.paged_evict(pool, b, b, pool.new_mass()),
                 lambda: hqmq.paged_store(pool, pool.K, pool.V, b)):
        with pytest.raises(_lib.HqmqError):
            call()


def test_a_cache_that_refuses_is_unchanged():
    cache, pool = hqmq.PagedKVCache(None, 8), make_pool()
    a, b = cache.add(2)
    cache.begin([a, b], [200, 64])                                       # 4 pages, 1 page
    assert cache.free_pages == 3
    for call, error in ((lambda: cache.begin([a], [300]), _lib.HqmqError), (lambda: cache.begin([a, a], [1, 1]), ValueError),
                        (lambda: cache.begin([7], [1]), KeyError), (lambda: cache.begin([a], [-1]), ValueError),
                        (lambda: cache.evict([a], keep=10), ValueError), (lambda: cache.drop([a, 9]), KeyError)):
        with pytest.raises(error):
            call()
    cache._pools[0], cache._mass[0] = pool, pool.new_mass()
    for kw, error in (({"first": -1}, ValueError), ({"last": -4}, ValueError), ({"first": 40, "last": 41}, ValueError)):
        with pytest.raises(error):
            cache.evict([a], keep=80, **kw)
    cache.begin([b], [128])                                              # one page left
    with pytest.raises(_lib.HqmqError):
        cache.evict([a], keep=80)                                        # wants two
    assert cache.free_pages == 1 and cache.length(a) == 200 and cache.length(b) == 192 and cache._step == ([b], [128])
    cache.drop([a, b])
    assert cache.free_pages == 8


def _args(pool, batch, G=2):
    a = _lib.PagedAttnArgs(struct_size=C.sizeof(_lib.PagedAttnArgs), q_dtype=_lib.BF16, o_dtype=_lib.BF16, r_qmax=7, softmax_scale=0.1)
    a.Q = a.O = a.plan_data = a.table_K = a.table_V = a.mass = 1 << 20
    a.K, a.V, a.plan = pool.K.c_struct(), pool.V.c_struct(), batch.plan
    return a


@pytest.mark.parametrize("change,code", [
    (dict(struct_size=8), -1), (dict(Q=None), -1), (dict(O=None), -1), (dict(plan_data=None), -1), (dict(table_K=None), -1),
    (dict(q_dtype=_lib.I32), -3), (dict(o_dtype=_lib.I8), -3), (dict(plan_data=(1 << 20) + 4), -4), (dict(r_qmax=15), -2),
    (dict(softcap=-1.0), -1), (dict(softcap=float("nan")), -1), (dict(softmax_scale=float("nan")), -1), (dict(softmax_scale=0.0), -1),
    (dict(softcap=2e4), -1), ({}, -5),
])
def test_abi_refuses_arguments(built_lib, change, code):
    pool = make_pool(outliers_K=True)
    a = _args(pool, hqmq.PagedBatch(pool, [[0, 1], [2]], [100, 50], [1, 1], n_heads=4))
    for k, v in change.items():
        setattr(a, k, v)
    L = _lib.lib()
    assert L.hqmq_paged_attn(C.byref(a), None, 0, None) == code
    assert (L.hqmq_paged_attn_workspace_bytes(C.byref(a)) == 0) == bool(change)


def test_abi_refuses_pools_of_another_kind(built_lib):
    pool = make_pool(outliers_K=True)
    b = hqmq.PagedBatch(pool, [[0, 1], [2]], [100, 50], [1, 1], n_heads=4)
    L = _lib.lib()
    for field, value, code in (("B", 63, -2), ("H", 4, -2), ("T_cap", 128, -2), ("scale_dtype", _lib.F32, -8), ("out_dtype", _lib.F32, -8)):
        a = _args(pool, b)
        setattr(a.K, field, value)
        assert L.hqmq_paged_attn(C.byref(a), None, 0, None) == code, field
    a = _args(pool, b)
    a.q_dtype = _lib.F32
    assert L.hqmq_paged_mass(C.byref(a), None, 0, None) == -8
    store = hqmq.PagedBatch(pool, [[0, 1]], [100], [1])                # without query heads
    assert L.hqmq_paged_attn(C.byref(_args(pool, store)), None, 0, None) == -1
    for change in (dict(page_tokens=32), dict(n_seqs=0), dict(d=96), dict(H_q=3)):
        a = _args(pool, b)
        for k, v in change.items():
            setattr(a.plan, k, v)
        assert L.hqmq_paged_attn(C.byref(a), None, 0, None) in (-2, -8)


def test_what_a_call_wrote_is_not_read_through_the_read_only_path():
    """The second kernel of a call may start while the first still runs: what that one writes (kept positions, partial results, scores,
    image scales) is no read-only memory, and a load that says so may be moved ahead of the wait."""
    csrc = os.path.join(os.path.dirname(hqmq.__file__), "csrc")
    written = re.compile(r"__ldg\((?:reinterpret_cast<[^()]*>\()?&?(?:[pe]\.)?(?:kept|parts|cta_parts|stats|scores|kmul|vmul|part|kimg|vimg|new_mass)\b")
    assert written.search("__ldg(kept + i)") and written.search("__ldg(reinterpret_cast<const float4*>(p.scores) + 1)")
    for name in os.listdir(csrc):
        if name.startswith(("paged", "attn_prefill")):
            assert not written.search(open(os.path.join(csrc, name)).read()), name


@pytest.mark.parametrize("H,G,window,q", [(8, 4, 0, 1), (2, 4, 0, 5), (8, 4, 4096, 1), (1, 1, 0, 1)])
def test_a_plan_with_room_has_the_ctas_of_the_lengths_it_may_serve(H, G, window, q):
    pages = 2100
    pool, rng = make_pool(pages, H=H), random.Random(1)
    tables = tables_for([131072, 64], 64, pages, rng)
    full = hqmq.PagedBatch(pool, tables, [131072, 64], [q, q], n_heads=H * G, window=window or None).plan
    short = hqmq.PagedBatch(pool, [t[:5] for t in tables], [300, 40], [q, q], n_heads=H * G, window=window or None, reserve_pages=2049)
    assert short.plan.dec_ctas >= full.dec_ctas and short.plan.ms_ctas >= full.ms_ctas
    none = hqmq.PagedBatch(pool, [t[:5] for t in tables], [300, 40], [q, q], n_heads=H * G, window=window or None).plan
    assert none.dec_ctas <= 148 // H and short.plan.dec_ctas * H <= 148 and short.plan.ms_ctas * H <= 148
    # and whatever the lengths, every tile lies in one warp's stretch
    p = _lib.PagedPlan.from_buffer_copy(short.plan)
    p.renew = 1
    for kv in ([300, 40], [5, 5], [131072, 64], [70000, 17]):
        host, *_ = short._lay_out(p, tables, kv, [q, q])
        w = host.numpy()
        lengths, own = [[n, q] for n in kv], [t[:-(-n // 64)] for t, n in zip(tables, kv)]
        for rows, unit, base, warp, total, ctas, per in ((q * G, p.dec_unit, p.dec_base, p.dec_warp, p.dec_tiles, p.dec_ctas, DEC_WARPS if p.dec_rows == 8 else DEC_WARPS_WIDE),
                                                        (p.ms_rows, p.ms_unit, p.ms_base, p.ms_warp, p.ms_tiles, p.ms_ctas, MASS_WARPS)):
            want = []
            for s in (0, 1):
                for r in range(0, q * G, rows):
                    lo, hi = keys_of(kv[s], q, G, window, r, min(q * G, r + rows))
                    want.append((s, r, lo // 16, -(-hi // 16)))
            check_flat(w, unit, base, warp, total, ctas, per, want, own, 64, lengths)


def test_prompts_whose_weights_have_no_room_are_attended_all_the_same(built_lib):
    n = 524288
    pool = make_pool(n // 64, H=8)
    table = [list(range(n // 64))]
    b = hqmq.PagedBatch(pool, table, [n], [n], n_heads=32)
    assert b.plan.no_mass == 1 and b.plan.ms_units == 0 and b.plan.ch_units == n // 64
    a = _args(pool, b)
    L = _lib.lib()
    assert L.hqmq_paged_mass(C.byref(a), None, 0, None) == -9 and L.hqmq_paged_mass_workspace_bytes(C.byref(a)) == 0
    assert L.hqmq_paged_attn_workspace_bytes(C.byref(a)) > 0
    # (the room of a batch that is renewed counts as well)
    b = hqmq.PagedBatch(pool, [[0]], [40], [32], n_heads=16, reserve_pages=1 << 24)
    assert b.plan.no_mass == 0
    b = hqmq.PagedBatch(pool, [[0]], [40], [32], n_heads=128, reserve_pages=1 << 24)
    assert b.plan.no_mass == 1
    # (the last tokens of the same prompt have weights)
    assert hqmq.PagedBatch(pool, table, [n], [32], n_heads=32).plan.no_mass == 0


def test_a_batch_keeps_its_lengths_when_the_callers_arrays_change():
    pool = make_pool()
    kv, q, tables = np.array([100, 90], np.int32), torch.tensor([1, 2], dtype=torch.int32), np.array([[1, 2], [3, 2]], np.int32)
    b = hqmq.PagedBatch(pool, tables, kv, q)
    kv += 40
    q.zero_()
    tables[1, 1] = 5
    assert b.kv_lens.tolist() == [100, 90] and b.q_lens.tolist() == [1, 2]
    assert not b.stores_alone()                                          # both write page 2, as the plan on the device does


@pytest.mark.parametrize("window", [1 << 31, (1 << 32) + 5, 1 << 40])
def test_a_window_wider_than_any_sequence_is_no_window(window):
    pool = make_pool()
    data = [hqmq.PagedBatch(pool, [[1, 2, 3]], [150], [60], n_heads=4, window=w) for w in (None, window)]
    assert torch.equal(data[0].data, data[1].data) and data[1].plan.window == 1 << 30


@pytest.mark.parametrize("room", [-1, (1 << 24) + 1, (1 << 32) + 8])
def test_rooms_that_no_plan_has_are_refused(room):
    with pytest.raises(ValueError):
        hqmq.PagedBatch(make_pool(), [[1]], [50], [1], n_heads=4, reserve_pages=room)


def test_layers_of_unlike_pools_have_batches_of_their_own():
    cache = hqmq.PagedKVCache(None, 8)
    cache._pools.update({0: make_pool(8, H=2, d=128), 1: make_pool(8, H=2, d=64), 2: make_pool(8, H=2, d=128), 3: make_pool(8, H=1, d=64)})
    a, = cache.add()
    cache.begin([a], [100])
    got = [(cache.batch(layer, 4), cache.batch(layer)) for layer in range(4)]
    for layer, pair in enumerate(got):
        for b in pair:
            pool = cache.pool(layer)
            assert (b.d_head, b.H_kv, b.device, b.plan.d, b.plan.H_kv) == (pool.d_head, pool.H_kv, pool.device, pool.d_head, pool.H_kv)
    assert got[0][0] is got[2][0] and got[0][1] is got[2][1] and got[0][0] is not got[1][0]


def test_a_cache_whose_call_fails_half_way_loses_no_page():
    cache = hqmq.PagedKVCache(None, 16)
    cache._pools.update({0: make_pool(16, d=128), 1: make_pool(16, d=64)})
    cache._mass.update({layer: pool.new_mass() for layer, pool in cache._pools.items()})
    a, b = cache.add(2)
    cache.begin([a, b], [200, 300])
    state = lambda: (list(cache._free), {i: list(t) for i, t in cache._table.items()}, dict(cache._len), cache._step)
    before = state()
    with pytest.raises(_lib.HqmqError):                                  # (these pools are no CUDA memory)
        cache.evict([a, b], keep=100)
    assert state() == before

    class Busy:                                                          # (a copy to the device inside a graph's capture)
        device = "cpu"

        def __setitem__(self, *_):
            raise RuntimeError("capturing")

    cache._mass[1] = Busy()
    for call in (lambda: cache.begin([a], [200]), lambda: cache.evict([b], keep=100)):
        with pytest.raises(RuntimeError):
            call()
        assert state() == before
    assert cache.free_pages == 16 - 4 - 5


def _checked_cache(lens, updated=True):
    cache = hqmq.PagedKVCache(None, 12)
    pool = cache._pools[0] = make_pool(12, outliers_K=True, outliers_V=True, out_cap=8)
    for pk in (pool.K, pool.V):                                          # (what recycled pages may hold)
        pk.pages("rs").fill_(float("nan"))
        pk.pages("out_count").fill_(1 << 20)
    ids = cache.add(len(lens))
    cache.begin(ids, lens)
    for i in ids:
        for k, p in enumerate(cache._table[i]):
            for pk in (pool.K, pool.V):
                pk.pages("rs")[p, :, :min(64, lens[ids.index(i)] - 64 * k)] = 1.0
                pk.pages("out_count")[p] = 8
    if updated:
        cache._updated = {0}
    return cache, pool, ids


@pytest.mark.parametrize("lens,token", [([63], 62), ([1, 200], 199), ([64, 65], 64), ([130], 5)])
@pytest.mark.parametrize("plane", ["K", "V"])
def test_check_looks_at_every_token_that_is_held(lens, token, plane):
    cache, pool, ids = _checked_cache(lens)
    cache.check()
    getattr(pool, plane).pages("rs")[cache._table[ids[-1]][token // 64], 1, token % 64] = float("nan")
    with pytest.raises(_lib.HqmqError, match="bounded wait"):
        cache.check()
    cache.drop([ids[-1]])
    cache.check()


@pytest.mark.parametrize("plane", ["K", "V"])
def test_check_forgets_the_overflows_of_pages_that_are_free(plane):
    cache, pool, (a, b) = _checked_cache([100, 40])
    getattr(pool, plane).pages("out_count")[cache._table[b][0], 1] = 9
    with pytest.raises(_lib.HqmqError, match="overflowed"):
        cache.check()
    with pytest.raises(_lib.HqmqError, match="overflowed"):
        pool.check()
    cache.drop([b])
    cache.check()
    pool.check(cache._table[a])
    cache.drop([a])
    cache.check()


def test_check_in_the_middle_of_a_step():
    cache, pool, (a, b) = _checked_cache([100, 40])
    cache.begin([a, b], [60, 1])                                         # a page of an earlier life, and rows of one
    cache.check()
    cache._updated.add(0)
    with pytest.raises(_lib.HqmqError):
        cache.check()
