"""Plain 64-bit forms of the batched serving operators, for their tests, and
the device-side helpers around the calls."""
import math

import numpy as np
import torch

import vkv
from gpu_util import dev, stream_ptr

TORCH = {vkv.F32: torch.float32, vkv.F16: torch.float16, vkv.BF16: torch.bfloat16}
CODES = {vkv.E4M3: torch.float8_e4m3fn, vkv.I8: torch.int8}
TOP = {vkv.E4M3: 448.0, vkv.I8: 127.0}


def half_step(dtype):
    return torch.finfo(TORCH[dtype]).eps / 2


# ---- page map ----
def map_reference(old, new, page, n_pages, table, free, n_free, max_tokens):
    """(table, free, n_free, lens, cu, slots, positions, status) by loops over requests, entries and tokens"""
    table, free = table.copy(), free.copy()
    cap = table.shape[1] * page
    none = (table.copy(), free.copy(), n_free, list(old), [0] * (len(old) + 1), [-1] * max_tokens, [-1] * max_tokens)
    if not 0 <= n_free <= n_pages or any(not 0 <= x <= cap for x in list(old) + list(new)):
        return none + (2,)
    held = [-(-x // page) for x in old]
    want = [-(-x // page) for x in new]
    back = [int(table[r, e]) for r in range(len(old)) for e in range(want[r], held[r])]
    if sum(max(0, b - a) for a, b in zip(old, new)) > max_tokens or n_free + len(back) > n_pages:
        return none + (2,)
    if any(not 0 <= p < n_pages for p in back):
        return none + (2,)
    if sum(max(0, w - h) for h, w in zip(held, want)) > n_free + len(back):
        return none + (1,)
    for p in back:
        free[n_free] = p
        n_free += 1
    cu, slots, positions = [0], [], []
    for r in range(len(old)):
        for e in range(held[r], want[r]):
            n_free -= 1
            table[r, e] = free[n_free]
        for pos in range(old[r], new[r]):
            slots.append(int(table[r, pos // page]) * page + pos % page)
            positions.append(pos)
        cu.append(len(slots))
    pad = [-1] * (max_tokens - len(slots))
    return table, free, n_free, list(new), cu, slots + pad, positions + pad, 0


class Map:
    """Device arrays of a page map and the call."""

    def __init__(self, page, n_pages, n_req, stride, free=None, n_free=None, table=None):
        i32 = dict(dtype=torch.int32, device=dev())
        self.page, self.n_pages, self.n_req, self.stride = page, n_pages, n_req, stride
        self.table = torch.full((n_req, stride), -7, **i32) if table is None else torch.as_tensor(table, **i32)
        self.free = torch.as_tensor(np.arange(n_pages)[::-1].copy() if free is None else free, **i32)
        self.n_free = torch.tensor([n_pages if n_free is None else n_free], **i32)
        self.lens = torch.zeros(n_req, **i32)
        self.cu = torch.full((n_req + 1,), -9, **i32)
        self.status = torch.full((1,), -9, **i32)

    def room(self, max_tokens):
        i32 = dict(dtype=torch.int32, device=dev())
        self.max_tokens = max_tokens
        self.slots = torch.full((max_tokens,), -9, **i32)
        self.positions = torch.full((max_tokens,), -9, **i32)

    def call(self, new, n_free_out=None):
        """in place: lengths and stack size where they are"""
        vkv.page_map(self.lens.data_ptr(), new.data_ptr(), self.n_req, self.page, self.n_pages, self.table.data_ptr(),
                     self.stride, self.free.data_ptr(), self.n_free.data_ptr(),
                     (self.n_free if n_free_out is None else n_free_out).data_ptr(), self.max_tokens,
                     self.lens.data_ptr(), self.cu.data_ptr(), self.slots.data_ptr(), self.positions.data_ptr(),
                     self.status.data_ptr(), hip_stream=stream_ptr())


# ---- pages ----
def nearest(x, code):
    """value of the nearest code, ties to even, of float64 values in units of the scale"""
    if code == vkv.I8:
        return np.clip(np.rint(np.nan_to_num(x, nan=0.0, posinf=127, neginf=-127)), -127, 127)
    with np.errstate(all="ignore"):
        e = np.maximum(np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -40))), -6)
        step = np.exp2(e - 3)
        return np.where(np.isfinite(x), np.rint(x / step) * step, np.nan)


def scale_for(amax, code):
    """the least power of two, 2^-100 to 2^120, that holds amax"""
    e = -100
    if amax > 0:
        m, x = math.frexp(amax / TOP[code])
        e = x - 1 if m == 0.5 else x
    return 2.0 ** min(max(e, -100), 120)


class Pool:
    """Pages on the device, and the values they should hold by token."""

    def __init__(self, code, n_pages, page, heads, dim, n_layers=1, fill=None):
        self.code, self.n_pages, self.page, self.heads, self.dim, self.n_layers = code, n_pages, page, heads, dim, n_layers
        shape = (n_layers, n_pages, heads, page * dim)
        # what a fresh allocation may hold: NaN codes and scales
        self.codes = [torch.full(shape, 0x7f if fill is None else fill, dtype=torch.uint8, device=dev()) for _ in "kv"]
        self.scale = [torch.full(shape[:3], float("nan"), dtype=torch.float32, device=dev()) for _ in "kv"]
        self.desc = vkv.Pages(self.codes[0].data_ptr(), self.codes[1].data_ptr(), self.scale[0].data_ptr(),
                              self.scale[1].data_ptr(), code, n_layers, n_pages, page, heads, dim)

    def append(self, slots, k, v, dtype, layer=0, row_stride=0):
        vkv.pages_append(self.desc, layer, slots.data_ptr(), slots.numel(), dtype, k.data_ptr(), v.data_ptr(),
                         row_stride=row_stride, hip_stream=stream_ptr())

    def read(self, layer=0):
        """K and V codes' values [page][head][token][dim] and the scales, float64"""
        torch.cuda.synchronize()
        p, h, s, d = self.n_pages, self.heads, self.page, self.dim
        out = []
        for i in range(2):
            c = self.codes[i][layer].cpu().view(CODES[self.code]).double().numpy()
            if i == 0:
                c = c.reshape(p, h, s, d)
            else:   # [block][r][g][t][j] -> token 16 b + 4 g + j, dim 16 t + r
                c = c.reshape(p, h, s // 16, 16, 4, d // 16, 4).transpose(0, 1, 2, 4, 6, 5, 3).reshape(p, h, s, d)
            out.append((c, self.scale[i][layer].cpu().double().numpy()))
        return out


class PoolModel:
    """The pages as the definition has them: codes and scales in float64, one page and head after the other."""

    def __init__(self, code, n_pages, page, heads, dim):
        self.code, self.page, self.heads, self.dim, self.n_pages = code, page, heads, dim, n_pages
        self.codes = [np.full((n_pages, heads, page, dim), np.nan if code == vkv.E4M3 else 127.0) for _ in "kv"]
        self.scale = [np.full((n_pages, heads), np.nan) for _ in "kv"]

    def append(self, slots, k, v):
        by_page = {}
        for i, s in enumerate(slots):
            if 0 <= s < self.n_pages * self.page:
                by_page.setdefault(int(s) // self.page, {})[int(s) % self.page] = i   # the last one counts
        for w, rows in enumerate((k, v)):
            rows = rows.reshape(len(slots), self.heads, self.dim).astype(np.float64)
            for page, got in by_page.items():
                for h in range(self.heads):
                    x = np.stack([rows[i, h] for i in got.values()])
                    need = scale_for(np.max(np.abs(np.where(np.isfinite(x), x, 0.0))), self.code)
                    codes, old = self.codes[w][page, h], self.scale[w][page, h]
                    to = need if 0 in got else max(need, old)
                    if 0 not in got and to > old:
                        codes[:] = nearest(codes * (old / to), self.code)
                    for off, i in got.items():
                        codes[off] = nearest(rows[i, h] / to, self.code)
                    self.scale[w][page, h] = to


# ---- attention ----
def attend(q, k, v, live, scale):
    """softmax(scale q k^T) v per head in float64; q [nq][H][D], k, v [n][Hk][D], live [nq][n]; zeros without a key.
    Also the largest sum of |scale q k| and the weighted sum of |v|, for tolerances."""
    nq, H, D = q.shape
    g = H // k.shape[1]
    out, mass, vmass = np.zeros((nq, H, D)), 0.0, np.zeros((nq, H, D))
    for h in range(H):
        kk, vv = k[:, h // g], v[:, h // g]
        for i in range(nq):
            on = live[i]
            if not on.any():
                continue
            s = scale * (kk[on] @ q[i, h])
            p = np.exp(s - s.max())
            p /= p.sum()
            out[i, h] = p @ vv[on]
            vmass[i, h] = p @ np.abs(vv[on])
            mass = max(mass, float(np.max(abs(scale) * (np.abs(kk[on]) @ np.abs(q[i, h])))))
    return out, mass, vmass


def attend_tolerance(mass, vmass, want, dtype, dim, n, vmax, p_step=0.0):
    """Elementwise bound.  A score's terms are off by 2^-22 (the pair of f16) and their sum in f32 by dim 2^-24, of
    their magnitudes' sum `mass`; its product with the scale and log2 e and the exponent's argument by 3 2^-24 more.
    An exponent off by ds changes the output by no more than 2 ds of the weighted |v|, which is at most vmax.  The
    weights are off by 2^-22 (or p_step, where they are rounded to the rows' type), the sums over n keys by n 2^-24
    at the most and twice (numerator, denominator); last the result's own rounding."""
    ds = mass * (2.0 ** -22 + (dim + 3) * 2.0 ** -24) * 1.45
    rel = 2 * ds + 2.0 ** -22 + p_step + 2 * n * 2.0 ** -24
    return rel * np.maximum(vmass, 1e-3 * vmax) + half_step(dtype) * np.abs(want) * (1 + rel) + 1e-30


def rows_on_device(x, dtype):
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to(dev()).to(TORCH[dtype])


def as64(t):
    return t.detach().cpu().double().numpy()
