"""Page map, append and attention of the paged 8-bit K/V pool on the GPU,
against loops and float64."""
import numpy as np
import pytest
import torch

import vkv
from gpu_util import dev, stream_ptr
from serve_util import (TORCH, Map, Pool, PoolModel, as64, attend, attend_tolerance, map_reference, rows_on_device)

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.as_tensor(np.asarray(x, dtype=np.int32)).to(dev())


def ints(t):
    return t.cpu().numpy().tolist()


# ---- page map ----
def random_step(rng, n_req, cap, most):
    old = rng.integers(0, cap + 1, n_req)
    kind = rng.integers(0, 4, n_req)
    new = np.where(kind == 0, np.minimum(old + 1, cap), np.where(kind == 1, rng.integers(0, cap + 1, n_req),
                   np.where(kind == 2, 0, old)))
    return old, np.where(new - old > most, old + 1, new).clip(0, cap)


@pytest.mark.parametrize("n_req,page,stride,most", [(1, 16, 1, 16), (3, 16, 5, 80), (64, 32, 7, 40), (1023, 16, 4, 3),
                                                    (1024, 64, 3, 100), (1025, 16, 6, 9), (2500, 128, 2, 30)])
def test_page_map_equals_the_loops(n_req, page, stride, most):
    rng = np.random.default_rng(n_req)
    for _ in range(3):
        old, new = random_step(rng, n_req, stride * page, most)
        held = -(-old // page)
        need = np.maximum(-(-new // page) - held, 0).sum()
        n_pages = int(held.sum() + need + rng.integers(0, 9)) + 1
        order = rng.permutation(n_pages)
        table = np.full((n_req, stride), -7)
        at = 0
        for r, h in enumerate(held):
            table[r, :h] = order[at:at + h]
            at += h
        free = np.concatenate([order[at:], np.full(at, -5)])
        total = int(np.maximum(new - old, 0).sum())
        m = Map(page, n_pages, n_req, stride, free=free, n_free=n_pages - at, table=table)
        m.lens.copy_(i32(old))
        m.room(total + int(rng.integers(0, 5)))
        want = map_reference(old, new, page, n_pages, table, free, n_pages - at, m.max_tokens)
        m.call(i32(new))
        got = (m.table, m.free, m.n_free, m.lens, m.cu, m.slots, m.positions, m.status)
        for g, w, name in zip(got, want, ("table", "free", "n_free", "lens", "cu", "slots", "positions", "status")):
            assert np.array_equal(g.cpu().numpy().reshape(-1), np.asarray(w).reshape(-1)), name


def test_page_map_with_many_tokens_is_the_same():
    """beyond 4096 new tokens the slots are a launch of their own"""
    page, stride = 16, 400
    old = [0, 17, 0, 5, 300, 6400]
    new = [5000, 17, 1, 4000, 0, 6400]
    rng = np.random.default_rng(5)
    held = [-(-x // page) for x in old]
    n_pages = 1500
    order = rng.permutation(n_pages)
    table = np.full((6, stride), -7)
    at = 0
    for r, h in enumerate(held):
        table[r, :h] = order[at:at + h]
        at += h
    free = np.concatenate([order[at:], np.zeros(at, int)])
    m = Map(page, n_pages, 6, stride, free=free, n_free=n_pages - at, table=table)
    m.lens.copy_(i32(old))
    m.room(9100)
    want = map_reference(old, new, page, n_pages, table, free, n_pages - at, 9100)
    m.call(i32(new))
    for g, w in zip((m.table, m.free, m.n_free, m.lens, m.cu, m.slots, m.positions, m.status), want):
        assert np.array_equal(g.cpu().numpy().reshape(-1), np.asarray(w).reshape(-1))


@pytest.mark.parametrize("n_req,page,stride,most", [(65, 16, 9, 100), (200, 32, 4, 90), (256, 16, 8, 12), (257, 16, 3, 40),
                                                    (4100, 16, 2, 3), (5000, 16, 3, 30)])
def test_page_map_of_larger_batches(n_req, page, stride, most):
    """each of the map's forms at its ends, with few and with many new tokens"""
    test_page_map_equals_the_loops(n_req, page, stride, most)


@pytest.mark.parametrize("what,status", [
    ("short", 1), ("short of one page", 1), ("negative old", 2), ("negative new", 2), ("beyond the table", 2), ("too many tokens", 2),
    ("stack beyond the pool", 2), ("stack below 0", 2), ("returns no page", 2), ("more returned than the stack holds", 2),
    ("huge", 2)])
@pytest.mark.parametrize("max_tokens", [40, 5000])
def test_page_map_that_does_not_fit_changes_nothing(what, status, max_tokens):
    page, stride, n_pages = 16, 8, 12
    old, new = [20, 3, 40], [22, 0, 55]
    table = np.full((3, stride), -7)
    table[0, :2], table[1, :1], table[2, :3] = [3, 4], [9], [0, 1, 2]
    free, n_free = np.array([5, 6, 7, 8, 10, 11] + [-5] * 6), 6
    if what == "short":
        n_free, new = 0, [22, 3, 128]
        status = 2 if max_tokens == 40 else 1      # 90 new tokens
    elif what == "short of one page":
        n_free, new = 1, [33, 3, 50]
    elif what == "negative old":
        old = [20, -3, 40]
    elif what == "negative new":
        new = [22, -1, 55]
    elif what == "beyond the table":
        new = [22, 0, 129]
    elif what == "too many tokens":
        old, new = ([0, 3, 40], [20, 20, 60]) if max_tokens == 40 else ([2 ** 31 - 1, 3, 40], [0, 0, 0])
    elif what == "stack beyond the pool":
        n_free = 13
    elif what == "stack below 0":
        n_free = -1
    elif what == "returns no page":
        table[1, 0] = 12
    elif what == "more returned than the stack holds":
        n_free, new = 12, [20, 0, 40]
    elif what == "huge":
        old, new = [2 ** 31 - 1] * 3, [-2 ** 31, 2 ** 31 - 1, 5]
    m = Map(page, n_pages, 3, stride, free=free, n_free=n_free, table=table)
    m.lens.copy_(i32(old))
    m.room(max_tokens)
    m.call(i32(new))
    assert ints(m.status) == [status]
    assert np.array_equal(m.table.cpu().numpy(), table) and ints(m.free) == free.tolist() and ints(m.n_free) == [n_free]
    assert ints(m.lens) == old and ints(m.cu) == [0, 0, 0, 0]
    assert ints(m.slots) == [-1] * max_tokens and ints(m.positions) == [-1] * max_tokens


def test_page_map_over_a_life_of_requests():
    """sixty steps in place: no page is ever owned twice, none is lost"""
    rng = np.random.default_rng(3)
    page, stride, n_req, n_pages = 16, 12, 20, 90
    m = Map(page, n_pages, n_req, stride)
    m.room(600)
    lens = np.zeros(n_req, int)
    for _ in range(60):
        new = np.where(rng.random(n_req) < 0.15, 0, lens + rng.integers(0, 20, n_req)).clip(0, stride * page)
        m.call(i32(new))
        st = ints(m.status)[0]
        if st == 0:
            lens = new
        assert ints(m.lens) == lens.tolist()
        table, free = m.table.cpu().numpy(), ints(m.free)[:ints(m.n_free)[0]]
        owned = [int(p) for r in range(n_req) for p in table[r, :-(-lens[r] // page)]]
        assert sorted(owned + free) == list(range(n_pages))
        if st == 0:
            total = ints(m.cu)[-1]
            assert ints(m.slots)[total:] == [-1] * (600 - total)


# ---- append ----
CODES = [vkv.E4M3, vkv.I8]


def same_pages(pool, model, layer=0):
    for w, ((codes, scale), mc, ms) in enumerate(zip(pool.read(layer), model.codes, model.scale)):
        assert np.array_equal(scale, ms, equal_nan=True), ("scale", "kv"[w])
        bad = ~((codes == mc) | (np.isnan(codes) & np.isnan(mc)))
        assert not bad.any(), ("codes", "kv"[w], np.argwhere(bad)[:3].tolist(), codes[bad][:3], mc[bad][:3])


def wide_rows(rng, n, width, dtype):
    """values over many magnitudes, ties of the codes, zeros"""
    x = rng.standard_normal((n, width)) * np.exp2(rng.integers(-6, 7, (n, 1)))
    x[:, ::13] = np.exp2(rng.integers(-12, 4, x[:, ::13].shape)) * (rng.integers(8, 32, x[:, ::13].shape) + 0.5) / 16
    x[:, ::29] = 0
    return as64(rows_on_device(x, dtype))


@pytest.mark.parametrize("dtype", [vkv.F32, vkv.F16, vkv.BF16])
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("page,heads,dim", [(16, 8, 128), (32, 3, 64), (64, 1, 128), (128, 2, 64), (256, 1, 64)])
def test_append_equals_the_definition(page, heads, dim, code, dtype):
    """runs of many lengths: a prompt, single tokens that make a page's scale grow, a page begun again"""
    rng = np.random.default_rng(page + heads + dim + code + dtype)
    n_pages = 5
    pool, model = Pool(code, n_pages, page, heads, dim), PoolModel(code, n_pages, page, heads, dim)
    order = rng.permutation(n_pages - 1)          # one page stays untouched
    pos = 0
    for n in (page // 2 + 1, 1, 1, page, 1, 3, 16):
        slots = [int(order[(pos + i) // page % len(order)]) * page + (pos + i) % page for i in range(n)]
        pos += n
        k, v = (wide_rows(rng, n, heads * dim, dtype) for _ in range(2))
        pool.append(i32(slots), rows_on_device(k, dtype), rows_on_device(v, dtype), dtype)
        model.append(slots, k, v)
        same_pages(pool, model)


@pytest.mark.parametrize("code", CODES)
def test_append_skips_repeats_and_disorder(code):
    """-1 and slots outside the pool write nothing; a page's slots in any order; the last row of a slot counts"""
    rng = np.random.default_rng(8)
    page, heads, dim, n_pages = 32, 2, 64, 6
    pool, model = Pool(code, n_pages, page, heads, dim), PoolModel(code, n_pages, page, heads, dim)
    slots = [-1, 5, 3, 0, 3, 5, -1, n_pages * page, 2 ** 31 - 1, 70, 64, 70, 70, -2 ** 31, 33, 32] + [-1] * 3
    for _ in range(2):
        k, v = (wide_rows(rng, len(slots), heads * dim, vkv.F32) for _ in range(2))
        pool.append(i32(slots), rows_on_device(k, vkv.F32), rows_on_device(v, vkv.F32), vkv.F32)
        model.append(slots, k, v)
        same_pages(pool, model)
    # a run longer than the 256 tokens a work group looks at in one go
    slots = [96 + i % 32 for i in range(700)] + [128]
    k, v = (wide_rows(rng, len(slots), heads * dim, vkv.F32) for _ in range(2))
    pool.append(i32(slots), rows_on_device(k, vkv.F32), rows_on_device(v, vkv.F32), vkv.F32)
    model.append(slots, k, v)
    same_pages(pool, model)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("page,heads,dim,run", [(16, 3, 64, 50), (32, 2, 128, 7), (64, 1, 128, 300), (128, 1, 64, 700), (256, 1, 64, 90)])
def test_append_of_many_tokens(page, heads, dim, run, code):
    """more tokens than have a work group each: every page is begun with its slot 0, then runs begin and end anywhere in
    a page, twice; padding behind them"""
    rng = np.random.default_rng(run)
    n_pages, n = 0, 1300
    runs = []
    left = n
    while left:
        m = min(left, int(rng.integers(1, run + 1)))
        runs.append((int(rng.integers(0, page)), m))
        n_pages += -(-(runs[-1][0] + m) // page)
        left -= m
    order, slots, at = rng.permutation(n_pages), [], 0
    for first, m in runs:
        slots += [int(order[at + i // page]) * page + i % page for i in range(first, first + m)]
        at += -(-(first + m) // page)
    pool, model = Pool(code, n_pages, page, heads, dim), PoolModel(code, n_pages, page, heads, dim)
    for put in ([p * page for p in range(n_pages)], slots[:700], slots[700:] + [-1] * 30, slots):
        k, v = (wide_rows(rng, len(put), heads * dim, vkv.BF16) for _ in range(2))
        k, v = (rows_on_device(x, vkv.BF16) for x in (k, v))
        pool.append(i32(put), k, v, vkv.BF16)
        model.append(put, as64(k), as64(v))
        same_pages(pool, model)


@pytest.mark.parametrize("code", CODES)
def test_append_values_at_the_ends_of_the_range(code):
    """zeros, subnormals, the largest floats, infinities and NaN; a page's scale follows its finite values alone"""
    page, heads, dim = 16, 1, 64
    big = float(np.finfo(np.float32).max)
    specials = [0.0, -0.0, 1e-45, -1e-40, 1.2e-38, 2.0 ** -101, 2.0 ** -100 * 448, 2.0 ** -109, 448.0, 448.0 * 1.0001,
                127.0, 127.00001, 1.0, big, -big, float("inf"), float("-inf"), float("nan"), 1e30, -3.5]
    pool, model = Pool(code, len(specials) + 1, page, heads, dim), PoolModel(code, len(specials) + 1, page, heads, dim)
    for i, s in enumerate(specials):
        k = np.zeros((2, dim), np.float32)
        k[0, 0], k[0, 1], k[1, 5], k[1, 63] = s, 0.75, 1e-3, -s
        slots = [i * page, i * page + 1]
        pool.append(i32(slots), rows_on_device(k, vkv.F32), rows_on_device(k[::-1], vkv.F32), vkv.F32)
        model.append(slots, k, k[::-1])
        # and a token that may make the scale grow over what is there
        k = np.full((1, dim), 2.0 ** (i - 4), np.float32)
        pool.append(i32([i * page + 2]), rows_on_device(k, vkv.F32), rows_on_device(k, vkv.F32), vkv.F32)
        model.append([i * page + 2], k, k)
    same_pages(pool, model)


def test_append_rows_of_a_wider_array_and_another_layer():
    rng = np.random.default_rng(4)
    page, heads, dim, n_pages = 16, 2, 64, 3
    pool = Pool(vkv.E4M3, n_pages, page, heads, dim, n_layers=3)
    before = [c.clone() for c in pool.codes]
    qkv = rng.standard_normal((5, 4 * heads * dim)).astype(np.float32)
    t = rows_on_device(qkv, vkv.F16)
    k, v = t[:, 2 * heads * dim:], t[:, 3 * heads * dim:]
    pool.append(i32([16, 17, 18, 32, 33]), k, v, vkv.F16, layer=1, row_stride=t.shape[1])
    model = PoolModel(vkv.E4M3, n_pages, page, heads, dim)
    model.append([16, 17, 18, 32, 33], as64(k)[:, :heads * dim], as64(v))
    same_pages(pool, model, 1)
    for c, b in zip(pool.codes, before):
        assert torch.equal(c[0], b[0]) and torch.equal(c[2], b[2])


# ---- attention ----
def filled(rng, code, n_pages, page, heads, dim):
    """a pool of appended values, with NaN codes wherever nothing was appended"""
    pool = Pool(code, n_pages, page, heads, dim, fill=0x7f if code == vkv.E4M3 else 0x80)
    return pool


def requests(rng, pool, lens, stride):
    """append every request's tokens; the table, and K and V as the pages stand for them"""
    page, heads, dim = pool.page, pool.heads, pool.dim
    order = list(rng.permutation(pool.n_pages))
    table = np.full((len(lens), stride), -3)
    for r, n in enumerate(lens):
        for e in range(-(-n // page)):
            table[r, e] = order.pop()
        if n > 0:
            slots = [int(table[r, i // page]) * page + i % page for i in range(n)]
            k, v = (rng.standard_normal((n, heads * dim)) * np.exp2(rng.integers(-2, 3, (n, 1))) for _ in range(2))
            pool.append(i32(slots), rows_on_device(k, vkv.F32), rows_on_device(v, vkv.F32), vkv.F32)
    (kc, ks), (vc, vs) = pool.read()
    got = []
    for r, n in enumerate(lens):
        n = max(n, 0)
        ids = [int(table[r, i // page]) for i in range(n)]
        off = [i % page for i in range(n)]
        got.append(tuple((c[ids, :, off] * s[ids][..., None]).reshape(n, heads, dim) for c, s in ((kc, ks), (vc, vs))))
    return table, got


def check_attn(pool, table, lens, kv, H, dtype, window, rng, max_len=None, q_scale=1.0, scale=None, stride=None):
    dim = pool.dim
    scale = 1 / np.sqrt(dim) if scale is None else scale
    n = len(lens)
    q = as64(rows_on_device(rng.standard_normal((n, H * dim)) * q_scale, dtype))
    qd = rows_on_device(q, dtype)
    out = torch.full((n + 1, H * dim), 7.0, dtype=TORCH[dtype], device=dev())
    max_len = max(max(lens), 0) if max_len is None else max_len
    need = vkv.paged_attn_workspace(pool.desc, n, H, max_len)
    ws = torch.full((need + 64,), 0xff, dtype=torch.uint8, device=dev())
    t, le = i32(table), i32(lens)
    vkv.paged_attn(pool.desc, 0, t.data_ptr(), table.shape[1] if stride is None else stride, le.data_ptr(), n, max_len,
                   dtype, qd.data_ptr(), out.data_ptr(), H, scale, window, ws.data_ptr(), need, hip_stream=stream_ptr())
    got = as64(out)
    assert (got[n] == 7.0).all() and (ws[need:] == 0xff).all()
    for r in range(n):
        k, v = kv[r]
        live = np.ones((1, len(k)), bool)
        if window:
            live[0, :max(0, len(k) - window)] = False
        want, mass, vmass = attend(q[r].reshape(1, H, dim), k, v, live, scale)
        vmax = np.nanmax(np.abs(v)) if len(v) else 0.0
        tol = attend_tolerance(mass, vmass, want, dtype, dim, len(k), vmax)
        err = np.abs(got[r].reshape(1, H, dim) - want)
        assert (err <= tol).all(), (r, lens[r], err.max(), tol.max(), float((err / tol).max()))
    return out[:n]


@pytest.mark.parametrize("heads,group", [(8, 4), (2, 1), (1, 8), (3, 3), (1, 16), (2, 5), (1, 9)])
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype,dim,page", [(vkv.F32, 128, 16), (vkv.BF16, 64, 16), (vkv.F16, 128, 64)])
def test_paged_attn_lengths(heads, group, code, dtype, dim, page):
    rng = np.random.default_rng(heads * 100 + group + code + dim)
    lens = [0, 1, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129, 255, 256, 257, 300, 0]
    pool = Pool(code, sum(-(-n // page) for n in lens) + 1, page, heads, dim, fill=0x7f)
    table, kv = requests(rng, pool, lens, -(-300 // page))
    check_attn(pool, table, lens, kv, heads * group, dtype, 0, rng)


@pytest.mark.parametrize("window", [1, 7, 16, 31, 33, 200, 750])
@pytest.mark.parametrize("page", [16, 256])
def test_paged_attn_window(window, page):
    rng = np.random.default_rng(window)
    lens = [1, 16, 31, 32, 33, 64, 199, 200, 201, 333, 800, 1023]
    pool = Pool(vkv.E4M3, sum(-(-n // page) for n in lens), page, 2, 64, fill=0x7f)
    table, kv = requests(rng, pool, lens, -(-1023 // page))
    check_attn(pool, table, lens, kv, 8, vkv.F32, window, rng)


@pytest.mark.parametrize("lens,heads", [([5000], 1), ([9000, 1, 4097, 2049], 2), ([1025] * 40, 8)])
def test_paged_attn_long(lens, heads):
    """long rows, in chunks of every size, and a batch of more work groups than the card holds"""
    rng = np.random.default_rng(len(lens))
    page = 32
    pool = Pool(vkv.I8, sum(-(-n // page) for n in lens), page, heads, 128, fill=0x80)
    table, kv = requests(rng, pool, lens, -(-max(lens) // page) + 2)
    a = check_attn(pool, table, lens, kv, heads * 4, vkv.F32, 0, rng)
    b = check_attn(pool, table, lens, kv, heads * 4, vkv.F32, 0, np.random.default_rng(1), max_len=max(lens) + 40)
    assert torch.isfinite(a).all() and torch.isfinite(b).all()


def test_paged_attn_of_scores_far_apart():
    """scores of thousands: one key has all the weight"""
    rng = np.random.default_rng(12)
    pool = Pool(vkv.E4M3, 40, 16, 2, 128, fill=0x7f)
    table, kv = requests(rng, pool, [333, 17], 21)
    for q_scale, scale in ((300.0, None), (1e-30, None), (1.0, -0.1), (1.0, 0.0), (1e30, 1e-31)):
        check_attn(pool, table, [333, 17], kv, 8, vkv.F32, 0, rng, q_scale=q_scale, scale=scale)


def test_paged_attn_pages_of_very_different_scales():
    """the weights are scaled by a page's scale over the chunk's largest"""
    rng = np.random.default_rng(13)
    page, heads, dim, n = 16, 2, 64, 160
    pool = Pool(vkv.E4M3, 10, page, heads, dim, fill=0x7f)
    for p in range(10):
        k, v = rng.standard_normal((2, page, heads * dim))
        v *= 2.0 ** (9 * (p % 3) - 9)
        pool.append(i32(range(p * page, (p + 1) * page)), rows_on_device(k, vkv.F32), rows_on_device(v, vkv.F32), vkv.F32)
    (kc, ks), (vc, vs) = pool.read()
    k, v = ((c * s[..., None, None]).transpose(0, 2, 1, 3).reshape(n, heads, dim) for c, s in ((kc, ks), (vc, vs)))
    check_attn(pool, np.arange(10)[None], [n], [(k, v)], 8, vkv.F32, 0, rng)


def test_paged_attn_values_that_are_not_finite():
    """a NaN value that a row attends to makes its dim NaN, behind its last token or before its window it does nothing"""
    rng = np.random.default_rng(14)
    page, heads, dim = 16, 1, 64
    pool = Pool(vkv.E4M3, 4, page, heads, dim, fill=0x7f)
    k, v = rng.standard_normal((2, 64, dim)).astype(np.float32)
    v[20, 3], k[50, 7] = np.inf, np.nan
    pool.append(i32(range(64)), rows_on_device(k, vkv.F32), rows_on_device(v, vkv.F32), vkv.F32)
    (kc, ks), (vc, vs) = pool.read()
    k, v = ((c * s[..., None, None]).transpose(0, 2, 1, 3).reshape(64, heads, dim) for c, s in ((kc, ks), (vc, vs)))
    table = np.arange(4)[None].repeat(3, 0)
    check_attn(pool, table, [20, 17, 3], [(k[:n], v[:n]) for n in (20, 17, 3)], 4, vkv.F32, 0, rng)
    check_attn(pool, table, [50, 49, 40], [(k[:n], v[:n]) for n in (50, 49, 40)], 4, vkv.F32, 19, rng)
    q = rows_on_device(rng.standard_normal((2, 4 * dim)), vkv.F32)
    out = torch.empty_like(q)
    t, le = i32(table), i32([30, 60])
    vkv.paged_attn(pool.desc, 0, t.data_ptr(), 4, le.data_ptr(), 2, 64, vkv.F32, q.data_ptr(), out.data_ptr(), 4, 0.1,
                   hip_stream=stream_ptr())
    out = out.view(2, 4, dim).isnan()
    assert out[0, :, 3].all() and out[0].sum() == 4
    assert out[1].all()


def test_paged_attn_of_bad_lengths_and_pages_gives_nan():
    rng = np.random.default_rng(15)
    pool = Pool(vkv.E4M3, 12, 16, 2, 64, fill=0x7f)
    table, kv = requests(rng, pool, [40, 40, 40], 6)
    table[1, 1] = 12
    for max_len in (41, 96):
        q = rows_on_device(rng.standard_normal((6, 4 * 64)), vkv.F32)
        out = torch.full_like(q, 7.0)
        t, le = i32(table[[0, 1, 2, 0, 1, 2]]), i32([40, 40, 97, -5, 16, 2 ** 31 - 1])
        ws = torch.empty(vkv.paged_attn_workspace(pool.desc, 6, 4, max_len), dtype=torch.uint8, device=dev())
        vkv.paged_attn(pool.desc, 0, t.data_ptr(), 6, le.data_ptr(), 6, max_len, vkv.F32, q.data_ptr(), out.data_ptr(), 4,
                       0.1, 0, ws.data_ptr(), ws.numel(), hip_stream=stream_ptr())
        nan = out.isnan()
        assert nan[1].all() and nan[2].all() and nan[5].all()
        assert not nan[0].any() and not nan[4].any() and (out[3] == 0).all()
    # the page before the window is not looked at
    out.fill_(7.0)
    t, le = i32(table[[1]] * 0 + np.where(np.arange(6) == 0, -1, table[0])), i32([40])
    vkv.paged_attn(pool.desc, 0, t.data_ptr(), 6, le.data_ptr(), 1, 96, vkv.F32, q.data_ptr(), out.data_ptr(), 4, 0.1, 8,
                   ws.data_ptr(), ws.numel(), hip_stream=stream_ptr())
    assert torch.isfinite(out[0]).all()


def test_paged_attn_several_tokens_of_one_request():
    """rows over one table (stride 0), lengths rising: each sees its own past"""
    rng = np.random.default_rng(16)
    pool = Pool(vkv.E4M3, 9, 16, 2, 64, fill=0x7f)
    table, kv = requests(rng, pool, [130], 9)
    k, v = kv[0]
    lens = [126, 127, 128, 129, 130]
    check_attn(pool, table, lens, [(k[:n], v[:n]) for n in lens], 8, vkv.F32, 0, rng, stride=0)


def test_paged_attn_rows_of_wider_arrays():
    rng = np.random.default_rng(17)
    heads, dim, H = 2, 64, 6
    pool = Pool(vkv.I8, 9, 16, heads, dim, fill=0x80)
    table, kv = requests(rng, pool, [60, 20], 4)
    wide = rows_on_device(rng.standard_normal((2, 3 * H * dim)), vkv.F16)
    out = torch.full((2, 2 * H * dim), 7.0, dtype=torch.float16, device=dev())
    t, le = i32(table), i32([60, 20])
    vkv.paged_attn(pool.desc, 0, t.data_ptr(), 4, le.data_ptr(), 2, 64, vkv.F16, wide[:, H * dim:].data_ptr(),
                   out[:, H * dim:].data_ptr(), H, 0.125, q_stride=3 * H * dim, out_stride=2 * H * dim,
                   hip_stream=stream_ptr())
    packed = torch.empty(2, H * dim, dtype=torch.float16, device=dev())
    q = wide[:, H * dim:2 * H * dim].contiguous()
    vkv.paged_attn(pool.desc, 0, t.data_ptr(), 4, le.data_ptr(), 2, 64, vkv.F16, q.data_ptr(), packed.data_ptr(), H, 0.125,
                   hip_stream=stream_ptr())
    assert torch.equal(out[:, H * dim:], packed) and (out[:, :H * dim] == 7.0).all()


def test_pages_beyond_32_bits():
    """the last pages of a pool whose codes pass 4 GiB"""
    rng = np.random.default_rng(18)
    page, heads, dim = 256, 8, 128
    n_pages = 17000          # 4.46e9 bytes of K codes
    shape = (n_pages, heads, page * dim)
    codes = [torch.empty(shape, dtype=torch.uint8, device=dev()) for _ in "kv"]
    scale = [torch.empty(shape[:2], dtype=torch.float32, device=dev()) for _ in "kv"]
    desc = vkv.Pages(codes[0].data_ptr(), codes[1].data_ptr(), scale[0].data_ptr(), scale[1].data_ptr(), vkv.E4M3, 1, n_pages,
                     page, heads, dim)
    small = Pool(vkv.E4M3, 2, page, heads, dim)
    ids = [n_pages - 1, n_pages - 300]
    k, v = (rows_on_device(rng.standard_normal((300, heads * dim)), vkv.F32) for _ in range(2))
    for d, at in ((desc, ids), (small.desc, [1, 0])):
        s = i32([at[i // page] * page + i % page for i in range(300)])
        vkv.pages_append(d, 0, s.data_ptr(), 300, vkv.F32, k.data_ptr(), v.data_ptr(), hip_stream=stream_ptr())
    for w in range(2):
        for big, little in zip(ids, [1, 0]):
            n = page if big == ids[0] else 300 - page
            a, b = codes[w][big], small.codes[w][0, little]
            if w == 0 or n == page:
                assert torch.equal(a[:, :n * dim], b[:, :n * dim])
            assert torch.equal(scale[w][big], small.scale[w][0, little])
    q = rows_on_device(rng.standard_normal((1, 32 * dim)), vkv.F32)
    outs = []
    for d, at in ((desc, ids), (small.desc, [1, 0])):
        t, le, out = i32([at]), i32([300]), torch.empty_like(q)
        ws = torch.empty(vkv.paged_attn_workspace(d, 1, 32, 512), dtype=torch.uint8, device=dev())
        vkv.paged_attn(d, 0, t.data_ptr(), 2, le.data_ptr(), 1, 512, vkv.F32, q.data_ptr(), out.data_ptr(), 32, 0.1, 0,
                       ws.data_ptr(), ws.numel(), hip_stream=stream_ptr())
        outs.append(out)
    assert torch.equal(*outs) and torch.isfinite(outs[0]).all()
