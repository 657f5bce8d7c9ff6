"""The operators of a server that answers many requests from one pool of 8-bit
K/V pages: in plain torch operations, and as the library's calls.

Kinds of case (the "kind" of a case dict):

  map       block tables, slot maps and positions of a step from the requests'
            lengths before and after it, pages taken from and returned to a
            free stack
  append    a step's new K/V rows into the pages: 8-bit codes with one
            power-of-two scale per page and kv head
  attn      single-query attention with grouped heads over such pages
  prompt    causal attention of several prompts packed one behind the other
  logprobs  log probability of given tokens, entropy of the row and its
            likeliest tokens

Page layout (codes, one byte each; P pages of S tokens, Hk kv heads, D dims):
K is [P][Hk][S][D].  V is stored by blocks of 16 tokens with the token
innermost: token 16 b + 4 g + j, dim 16 t + r is at [P][Hk][b][r][g][t][j].
A code c of page p and head h stands for c * scale[p][h].
"""
import math
import os
import random
import sys

import torch

own = False

if os.path.join(os.getcwd(), "voxtral.cpp_amd") not in sys.path:
    sys.path.insert(0, os.path.join(os.getcwd(), "voxtral.cpp_amd"))

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
CODES = {"e4m3": torch.float8_e4m3fn, "i8": torch.int8}
# largest code of a format as m * 2^x with m in [0.5, 1), as frexp gives it
TOP = {"e4m3": (0.875, 9), "i8": (0.9921875, 7)}
E_MIN, E_MAX = -100, 120   # exponents of a scale
INF = float("inf")


def listed():
    return [
        # a decode step of a full small batch: every request grows by a token, the smallest call there is
        dict(name="map_decode_32", kind="map", rows=32, page=16, stride=512, max_new=1, done=0.05, room=64, mix=1),
        # a step that admits prompts, rolls some requests back and releases others
        dict(name="map_mixed_401", kind="map", rows=401, page=16, stride=512, max_new=509, done=0.1, room=65536, mix=2),
        # the decode step's K/V rows of one layer, as the decoder's products leave them
        dict(name="append_decode_32", kind="append", dtype="f32", kv="e4m3", page=16, kv_heads=8, head_dim=128,
             tokens=32, run=1, mix=3),
        # a step that prefills several prompts at once, ragged, into larger pages
        dict(name="append_prompts_4099", kind="append", dtype="bf16", kv="i8", page=64, kv_heads=8, head_dim=128,
             tokens=4099, run=733, mix=4),
        # one live session whose window is the decoder's full 8192
        dict(name="attn_1x8192", kind="attn", dtype="f32", kv="e4m3", page=16, heads=32, kv_heads=8, head_dim=128,
             rows=1, max_len=8192, window=0, mix=5),
        # a loaded server: lengths from one token to the window, some rows of the batch unused
        dict(name="attn_64_ragged", kind="attn", dtype="bf16", kv="e4m3", page=16, heads=32, kv_heads=8, head_dim=128,
             rows=64, max_len=8192, window=0, mix=6),
        # a model without grouped heads, short sessions, a sliding window
        dict(name="attn_131_heads_i8", kind="attn", dtype="f16", kv="i8", page=32, heads=32, kv_heads=32, head_dim=64,
             rows=131, max_len=1500, window=750, mix=7),
        # the prompt every session starts with
        dict(name="prompt_38", kind="prompt", dtype="f32", heads=32, kv_heads=8, head_dim=128, seqs=1, max_len=38,
             window=0, mix=8),
        # a step that admits several sessions with their histories
        dict(name="prompt_13_ragged", kind="prompt", dtype="f32", heads=32, kv_heads=8, head_dim=128, seqs=13,
             max_len=1021, window=0, mix=9),
        # a long history in one piece
        dict(name="prompt_8192_bf16", kind="prompt", dtype="bf16", heads=32, kv_heads=8, head_dim=128, seqs=1,
             max_len=8192, window=0, mix=10),
        # a token's confidence in a live session
        dict(name="logprobs_1", kind="logprobs", dtype="f32", rows=1, vocab=131072, top=5, mix=11),
        # rescoring a transcript: a row for each of its tokens
        dict(name="logprobs_251_bf16", kind="logprobs", dtype="bf16", rows=251, vocab=131072, top=20, mix=12),
    ]


def _log(rng, a, b):
    return max(a, min(b, int(round(math.exp(rng.uniform(math.log(a), math.log(b + 0.5)))))))


def draw(rng):
    kind = rng.choice(["map", "append", "attn", "attn", "prompt", "prompt", "logprobs"])
    c = dict(kind=kind, mix=rng.randrange(1 << 20))
    if kind == "map":
        c.update(rows=_log(rng, 1, 401), page=rng.choice([16, 32, 64, 128]), max_new=_log(rng, 1, 509),
                 done=rng.choice([0.0, 0.05, 0.2]))
        c.update(stride=8192 // c["page"], room=_log(rng, 64, 65536))
        return c
    c.update(dtype=rng.choice(list(TYPES)))
    if kind == "logprobs":
        c.update(rows=_log(rng, 1, 251), vocab=rng.choice([131072, _log(rng, 33, 131071), _log(rng, 1024, 131071)]),
                 top=rng.randint(0, 32))
        return c
    kv_heads, group = rng.choice([(8, 4), (8, 4), (32, 1), (2, 8), (4, 3), (1, 16), (5, 2)])
    c.update(kv_heads=kv_heads, head_dim=rng.choice([64, 128]))
    if kind == "append":
        c.update(kv=rng.choice(list(CODES)), page=rng.choice([16, 32, 64, 128]), tokens=_log(rng, 1, 4099),
                 run=_log(rng, 1, 733))
        return c
    c.update(heads=kv_heads * group, window=rng.choice([0, 0, rng.randint(1, 1000)]))
    if kind == "attn":
        c.update(kv=rng.choice(list(CODES)), page=rng.choice([16, 32, 64, 128]), max_len=_log(rng, 1, 8192))
        c.update(rows=_log(rng, 1, min(131, max(1, (64 * 8192 * 8) // (c["max_len"] * kv_heads)))))
        return c
    c.update(max_len=_log(rng, 1, 4096))
    c.update(seqs=_log(rng, 1, min(64, max(1, 8192 // c["max_len"]))))
    return c


def _lens(case, n, most):
    """Lengths of a batch: the longest and the shortest there may be, the others spread; the same for every seed."""
    r = random.Random(case["mix"])
    lens = [r.randint(max(1, most // 16), most) for _ in range(n)]
    lens[0] = most
    if n > 2:
        lens[1] = 1
    if n > 8 and case["kind"] == "attn":
        lens[2] = 0   # an unused row of a batch of fixed size
    r.shuffle(lens)
    return lens


def _map_lens(case):
    """Lengths before and after a step."""
    r = random.Random(case["mix"])
    cap = case["stride"] * case["page"]
    old, new, room = [], [], case["room"]
    for _ in range(case["rows"]):
        if r.random() < case["done"]:      # released, or rolled back by a few tokens
            a = r.randint(1, cap // 8)
            old.append(a)
            new.append(0 if r.random() < 0.5 else max(0, a - r.randint(1, 40)))
            continue
        grow = 1 if r.random() < 0.7 else r.randint(1, case["max_new"])
        a = 0 if grow > 1 else r.randint(0, cap // 8)
        grow = min(grow, room)
        room -= grow
        old.append(a)
        new.append(a + grow)
    return old, new


def _runs(case):
    """Token counts of an append's requests, and the lengths they are appended at."""
    r = random.Random(case["mix"])
    counts, left = [], case["tokens"]
    while left:
        n = min(left, r.randint(1, case["run"]))
        counts.append(n)
        left -= n
    return [(r.randint(0, 3 * case["page"]), n) for n in counts]


def _rows(g, n, heads, dim, dtype):
    """Projected rows: unit spread, a few channels of a head several times larger, as trained keys and values have them."""
    x = torch.randn(n, heads, dim, generator=g, device="cuda")
    gain = torch.exp(0.3 * torch.randn(heads, dim, generator=g, device="cuda"))
    gain[:, :: 31] *= 4
    return (x * gain).reshape(n, heads * dim).to(dtype)


def _pool(g, case, pages):
    """K and V pages as earlier appends left them, with their scales."""
    h, s, d, kv = case["kv_heads"], case["page"], case["head_dim"], case["kv"]
    got = []
    for _ in range(2):
        codes = torch.empty(pages, h, s * d, dtype=CODES[kv], device="cuda")
        scale = torch.empty(pages, h, dtype=torch.float32, device="cuda")
        for at in range(0, pages, 4096):
            x = torch.randn(min(4096, pages - at), h, s * d, generator=g, device="cuda")
            x *= torch.exp(0.5 * torch.randn(x.shape[0], h, 1, generator=g, device="cuda"))
            e = _exponent(x.abs().amax(2), kv)
            codes[at:at + 4096] = _to_codes(x * torch.exp2(-e.float())[..., None], kv)
            scale[at:at + 4096] = torch.exp2(e.float())
        got += [codes, scale]
    return got


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 13)
    kind = case["kind"]
    st = dict(case=case)
    i32 = dict(dtype=torch.int32, device="cuda")
    if kind == "map":
        old, new = _map_lens(case)
        page, stride, rows = case["page"], case["stride"], case["rows"]
        held = [-(-n // page) for n in old]
        pages = sum(held) + sum(max(0, -(-n // page) - h) for n, h in zip(new, held)) + 37
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        table = torch.full((rows, stride), -1, **i32)
        at = 0
        for r, n in enumerate(held):
            table[r, :n] = order[at:at + n]
            at += n
        free = torch.zeros(pages, **i32)
        free[:pages - at] = order[at:]
        room = max(1, sum(max(0, b - a) for a, b in zip(old, new)) + 5)
        st.update(old=torch.tensor(old, **i32), new=torch.tensor(new, **i32), table=table, free=free,
                  n_free=torch.tensor([pages - at], **i32), n_free_out=torch.zeros(1, **i32), pages=pages, room=room,
                  lens=torch.zeros(rows, **i32), cu=torch.zeros(rows + 1, **i32), slots=torch.zeros(room, **i32),
                  positions=torch.zeros(room, **i32), status=torch.zeros(1, **i32))
        return st
    dtype = TYPES[case["dtype"]]
    if kind == "logprobs":
        n, v = case["rows"], case["vocab"]
        x = torch.empty(n, v, dtype=dtype, device="cuda")
        for at in range(0, n, 64):
            y = 2.5 * torch.randn(min(64, n - at), v, generator=g, device="cuda")
            # a decoder is sure of most tokens, and some ids are never to be said
            top = torch.randint(0, v, (y.shape[0], 3), generator=g, device="cuda")
            y.scatter_add_(1, top, torch.rand(y.shape[0], 3, generator=g, device="cuda") * 18)
            y[:, 1:max(2, v // 100):7] = -INF
            x[at:at + 64] = y.to(dtype)
        tokens = torch.randint(0, v, (n,), generator=g, device="cuda", dtype=torch.int32)
        tokens[::2] = x[::2].argmax(1).to(torch.int32)
        st.update(logits=x, tokens=tokens, logprob=torch.empty(n, device="cuda"), entropy=torch.empty(n, device="cuda"),
                  top_ids=torch.empty(n, case["top"], **i32), top_logprobs=torch.empty(n, case["top"], device="cuda"))
        return st
    h, d = case["kv_heads"], case["head_dim"]
    if kind == "append":
        runs, page = _runs(case), case["page"]
        need = [-(-(a + n) // page) for a, n in runs]
        pages = sum(need) + 3
        order = torch.randperm(pages, generator=g, device="cuda")
        slots, at = [], 0
        for (a, n), m in zip(runs, need):
            pos = torch.arange(a, a + n, device="cuda")
            slots.append(order[at:at + m][pos // page] * page + pos % page)
            at += m
        kc, ks, vc, vs = _pool(g, case, pages)
        st.update(slots=torch.cat(slots).to(torch.int32), k=_rows(g, case["tokens"], h, d, dtype),
                  v=_rows(g, case["tokens"], h, d, dtype), k_codes=kc, k_scale=ks, v_codes=vc, v_scale=vs, pages=pages)
        return st
    if kind == "attn":
        lens = _lens(case, case["rows"], case["max_len"])
        page = case["page"]
        stride = -(-case["max_len"] // page)
        need = [-(-n // page) for n in lens]
        pages = sum(need) + 3
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        table = torch.full((case["rows"], stride), -1, **i32)
        at = 0
        for r, m in enumerate(need):
            table[r, :m] = order[at:at + m]
            at += m
        kc, ks, vc, vs = _pool(g, case, pages)
        q = _rows(g, case["rows"], case["heads"], d, dtype)
        st.update(table=table, stride=stride, lens=torch.tensor(lens, **i32), q=q, out=torch.empty_like(q), k_codes=kc,
                  k_scale=ks, v_codes=vc, v_scale=vs, pages=pages)
        return st
    lens = _lens(case, case["seqs"], case["max_len"])
    cu = torch.tensor([0] + lens, device="cuda").cumsum(0).to(torch.int32)
    q = _rows(g, sum(lens), case["heads"], d, dtype)
    st.update(cu=cu, tokens=sum(lens), q=q, k=_rows(g, sum(lens), h, d, dtype), v=_rows(g, sum(lens), h, d, dtype),
              out=torch.empty_like(q))
    return st


# ---- plain forms ----

def _exponent(amax, kv):
    """The least e with amax <= largest code * 2^e, in the range of scales."""
    m, x = TOP[kv]
    f, e = torch.frexp(amax)
    e = e - x + (f > m).to(e.dtype)
    return torch.where(amax > 0, e, torch.full_like(e, E_MIN)).clamp(E_MIN, E_MAX)


def _to_codes(x, kv):
    """Values in units of the scale, to the nearest code (ties to even); what is not finite is NaN in e4m3, and in int8
    0 (NaN) or the largest code of its sign."""
    if kv == "e4m3":
        return torch.where(torch.isfinite(x), x, torch.full_like(x, float("nan"))).to(torch.float8_e4m3fn)
    return torch.nan_to_num(x, nan=0.0, posinf=127.0, neginf=-127.0).round().clamp(-127, 127).to(torch.int8)


def _v_rows(codes, s, d):
    """V pages [P, Hk, S D] as [P, Hk, S, D]."""
    p, h = codes.shape[:2]
    return codes.view(p, h, s // 16, 16, 4, d // 16, 4).permute(0, 1, 2, 4, 6, 5, 3).reshape(p, h, s, d)


def _v_stored(rows, s, d):
    p, h = rows.shape[:2]
    return rows.view(p, h, s // 16, 4, 4, d // 16, 16).permute(0, 1, 2, 6, 3, 5, 4).reshape(p, h, s * d)


def _map(st):
    c = st["case"]
    page, stride, pages, room = c["page"], c["stride"], st["pages"], st["room"]
    old, new, table = st["old"].long(), st["new"].long(), st["table"].long()
    held, want = (old + page - 1) // page, (new + page - 1) // page
    ret, take = (held - want).clamp(min=0), (want - held).clamp(min=0)
    grow = (new - old).clamp(min=0)
    n_in = st["n_free"].long()
    e = torch.arange(stride, device="cuda")[None]
    back, fresh = (e >= want[:, None]) & (e < held[:, None]), (e >= held[:, None]) & (e < want[:, None])
    cu = torch.cat([torch.zeros(1, dtype=torch.long, device="cuda"), grow.cumsum(0)])
    bad = ((old < 0) | (new < 0) | (old > stride * page) | (new > stride * page)).any() | (cu[-1] > room)
    bad = bad | (n_in < 0) | (n_in + ret.sum() > pages) | (back & ((table < 0) | (table >= pages))).any()
    short = take.sum() > n_in + ret.sum()
    good = ~(bad | short)
    # returned pages go on the stack in the order of requests and entries, taken ones come off its top
    at = n_in + (ret.cumsum(0) - ret)[:, None] + e - want[:, None]
    free = torch.cat([st["free"].long(), torch.zeros(1, dtype=torch.long, device="cuda")])
    free = free.scatter(0, torch.where(back & good, at, pages).reshape(-1), table.reshape(-1))[:pages]
    top = n_in + ret.sum()
    at = top - 1 - ((take.cumsum(0) - take)[:, None] + e - held[:, None])
    table = torch.where(fresh & good, free[at.clamp(0, pages - 1)], table)
    cu = torch.where(good, cu, 0)
    t = torch.arange(room, device="cuda")
    r = (torch.searchsorted(cu, t, right=True) - 1).clamp(max=c["rows"] - 1)
    pos = (old[r] + t - cu[r]).clamp(max=stride * page - 1)
    used = t < cu[-1]
    slots = torch.where(used, table[r, (pos // page).clamp(min=0)] * page + pos % page, -1)
    return dict(table=table.int(), free=torch.where(good, free, st["free"].long()).int(),
                n_free=torch.where(good, top - take.sum(), n_in).int(), lens=torch.where(good, new, old).int(),
                cu=cu.int(), slots=slots.int(), positions=torch.where(used, pos, -1).int(),
                status=torch.where(bad, 2, torch.where(short, 1, 0)).reshape(1).int())


def _append_one(st, x, codes, scale, is_v):
    c = st["case"]
    s, d, h, kv, pages = c["page"], c["head_dim"], c["kv_heads"], c["kv"], st["pages"]
    slot = st["slots"].long()
    page, off = slot // s, slot % s
    x = x.float().view(-1, h, d)
    amax = torch.where(torch.isfinite(x), x, torch.zeros_like(x)).abs().amax(2)
    need = _exponent(amax, kv).long()
    new = torch.full((pages, h), E_MIN, dtype=torch.long, device="cuda")
    new = new.scatter_reduce(0, page[:, None].expand(-1, h), need, "amax")
    written = torch.zeros(pages * s, dtype=torch.bool, device="cuda").index_fill(0, slot, True).view(pages, s)
    touched, fresh = written.any(1)[:, None], written[:, :1]
    old = torch.frexp(scale)[1].long() - 1
    e = torch.where(touched, torch.where(fresh, new, torch.maximum(old, new)), old)
    rows = (_v_rows(codes, s, d) if is_v else codes.view(pages, h, s, d))
    grown = (touched & ~fresh & (e > old))[..., None, None] & ~written[:, None, :, None]
    moved = _to_codes(rows.float() * torch.exp2((old - e).float())[..., None, None], kv)
    rows = torch.where(grown, moved.view(torch.uint8), rows.contiguous().view(torch.uint8))
    mine = _to_codes(x * torch.exp2(-e[page].float())[..., None], kv).view(torch.uint8)
    rows = rows.transpose(1, 2).reshape(pages * s, h, d).index_copy(0, slot, mine)
    rows = rows.view(pages, s, h, d).transpose(1, 2).contiguous()
    out = _v_stored(rows, s, d) if is_v else rows.view(pages, h, s * d)
    return out.contiguous().view(CODES[kv]), torch.where(touched, torch.exp2(e.float()), scale)


def _append(st):
    kc, ks = _append_one(st, st["k"], st["k_codes"], st["k_scale"], False)
    vc, vs = _append_one(st, st["v"], st["v_codes"], st["v_scale"], True)
    return dict(k=kc, k_scale=ks, v=vc, v_scale=vs)


def _attend(q, k, v, live, scale):
    """softmax(scale q k^T) v over the keys that `live` leaves; zeros where it leaves none."""
    s = torch.matmul(q, k.transpose(-1, -2)) * scale
    s = torch.where(live, s, torch.full_like(s, -INF))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m > -INF, m, torch.zeros_like(m)))
    del s
    z = p.sum(-1, keepdim=True)
    return torch.matmul(p / torch.where(z > 0, z, torch.ones_like(z)), v)


def _attn(st):
    c = st["case"]
    s, d, h, n = c["page"], c["head_dim"], c["kv_heads"], c["rows"]
    ids = st["table"].long().clamp(min=0)
    k = st["k_codes"][ids].float() * st["k_scale"][ids][..., None]
    v = _v_rows(st["v_codes"][ids].view(n * st["stride"], h, s * d), s, d).float()
    v = v * st["v_scale"][ids].view(-1, h, 1, 1)
    k = k.view(n, st["stride"], h, s, d).transpose(1, 2).reshape(n, h, -1, d)
    v = v.view(n, st["stride"], h, s, d).transpose(1, 2).reshape(n, h, -1, d)
    j = torch.arange(k.shape[2], device="cuda")[None]
    length = st["lens"].long()[:, None]
    live = j < length
    if c["window"]:
        live = live & (j >= length - c["window"])
    # codes behind the last token are anything: their rows do not count
    v = torch.where(live[:, None, :, None], v, torch.zeros_like(v))
    q = st["q"].float().view(n, h, -1, d)
    return _attend(q, k, v, live[:, None, None], 1 / math.sqrt(d)).reshape(n, -1).to(st["q"].dtype)


def _prompt(st):
    c = st["case"]
    d, h, n, m = c["head_dim"], c["kv_heads"], c["seqs"], c["max_len"]
    cu = st["cu"].long()
    j = torch.arange(m, device="cuda")
    live = j[None] < (cu[1:] - cu[:-1])[:, None]
    at = (cu[:-1, None] + j).clamp(max=max(0, st["tokens"] - 1))
    q = st["q"].float()[at].view(n, m, h, -1, d).permute(0, 2, 3, 1, 4)
    k, v = (st[w].float()[at].view(n, m, h, 1, d).permute(0, 2, 3, 1, 4) for w in "kv")
    seen = j[None] <= j[:, None]
    if c["window"]:
        seen = seen & (j[None] > j[:, None] - c["window"])
    g = q.shape[2]
    k, v = k.expand(-1, -1, g, -1, -1).contiguous(), v.expand(-1, -1, g, -1, -1).contiguous()
    o = _attend(q, k, v, seen & live[:, None, None, None, :], 1 / math.sqrt(d))
    o = o.permute(0, 3, 1, 2, 4).reshape(n * m, -1)
    # each sequence's rows to their place: the others go behind the last one
    to = torch.where(live, at, st["tokens"]).reshape(-1)
    out = torch.zeros(st["tokens"] + 1, o.shape[1], dtype=o.dtype, device="cuda")
    return out.index_copy(0, to, o)[:-1].to(st["q"].dtype)


def _logprobs(st):
    x, top = st["logits"].float(), st["case"]["top"]
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    z = e.double().sum(1, keepdim=True)
    log_z = torch.log(z)
    shifted = torch.where(e > 0, x - m, torch.zeros_like(x))
    entropy = log_z - (e * shifted).double().sum(1, keepdim=True) / z
    token = st["tokens"].long()[:, None]
    logprob = (x.gather(1, token) - m).double() - log_z
    value, ids = torch.sort(x, dim=1, descending=True, stable=True)
    return dict(logprob=logprob[:, 0].float(), entropy=entropy[:, 0].float(), top_ids=ids[:, :top].int(),
                top_logprobs=((value[:, :top] - m).double() - log_z).float())


PLAIN = dict(map=_map, append=_append, attn=_attn, prompt=_prompt, logprobs=_logprobs)


# ---- the library's calls ----

def _own(st):
    import vkv
    c = st["case"]
    kind = c["kind"]
    stream = torch.cuda.current_stream().cuda_stream
    if kind == "map":
        vkv.page_map(st["old"].data_ptr(), st["new"].data_ptr(), c["rows"], c["page"], st["pages"],
                     st["table"].data_ptr(), c["stride"], st["free"].data_ptr(), st["n_free"].data_ptr(),
                     st["n_free_out"].data_ptr(), st["room"], st["lens"].data_ptr(), st["cu"].data_ptr(),
                     st["slots"].data_ptr(), st["positions"].data_ptr(), st["status"].data_ptr(), hip_stream=stream)
        return dict(table=st["table"], free=st["free"], n_free=st["n_free_out"], lens=st["lens"], cu=st["cu"],
                    slots=st["slots"], positions=st["positions"], status=st["status"])
    dtype = dict(f32=vkv.F32, f16=vkv.F16, bf16=vkv.BF16)[c["dtype"]]
    if kind == "logprobs":
        if "ws" not in st:
            st["ws"] = torch.empty(vkv.logprobs_workspace(c["rows"], c["vocab"], c["top"]), dtype=torch.uint8, device="cuda")
        vkv.logprobs(dtype, st["logits"].data_ptr(), c["rows"], c["vocab"], st["tokens"].data_ptr(),
                     st["logprob"].data_ptr(), st["entropy"].data_ptr(), c["top"], st["top_ids"].data_ptr(),
                     st["top_logprobs"].data_ptr(), st["ws"].data_ptr(), st["ws"].numel(), hip_stream=stream)
        return dict(logprob=st["logprob"], entropy=st["entropy"], top_ids=st["top_ids"], top_logprobs=st["top_logprobs"])
    scale = 1 / math.sqrt(c["head_dim"])
    if kind == "prompt":
        if "ws" not in st:
            st["ws"] = torch.empty(vkv.prompt_attn_workspace(dtype, c["seqs"], st["tokens"], c["kv_heads"], c["head_dim"]),
                                   dtype=torch.uint8, device="cuda")
        vkv.prompt_attn(dtype, st["q"].data_ptr(), st["k"].data_ptr(), st["v"].data_ptr(), st["cu"].data_ptr(),
                        c["seqs"], st["tokens"], c["heads"], c["kv_heads"], c["head_dim"], scale, c["window"],
                        st["out"].data_ptr(), st["ws"].data_ptr(), st["ws"].numel(), hip_stream=stream)
        return st["out"]
    if "desc" not in st:
        st["desc"] = vkv.Pages(st["k_codes"].data_ptr(), st["v_codes"].data_ptr(), st["k_scale"].data_ptr(),
                               st["v_scale"].data_ptr(), dict(e4m3=vkv.E4M3, i8=vkv.I8)[c["kv"]], 1, st["pages"],
                               c["page"], c["kv_heads"], c["head_dim"])
    if kind == "append":
        vkv.pages_append(st["desc"], 0, st["slots"].data_ptr(), c["tokens"], dtype, st["k"].data_ptr(),
                         st["v"].data_ptr(), hip_stream=stream)
        return dict(k=st["k_codes"], k_scale=st["k_scale"], v=st["v_codes"], v_scale=st["v_scale"])
    if "ws" not in st:
        st["ws"] = torch.empty(vkv.paged_attn_workspace(st["desc"], c["rows"], c["heads"], c["max_len"]),
                               dtype=torch.uint8, device="cuda")
    vkv.paged_attn(st["desc"], 0, st["table"].data_ptr(), st["stride"], st["lens"].data_ptr(), c["rows"], c["max_len"],
                   dtype, st["q"].data_ptr(), st["out"].data_ptr(), c["heads"], scale, c["window"],
                   st["ws"].data_ptr(), st["ws"].numel(), hip_stream=stream)
    return st["out"]


def run(state):
    if own:
        return _own(state)
    return PLAIN[state["case"]["kind"]](state)


def work(case):
    kind = case["kind"]
    if kind == "map":
        old, new = _map_lens(case)
        s = case["page"]
        tokens = sum(max(0, b - a) for a, b in zip(old, new))
        moved = sum(abs(-(-a // s) - -(-b // s)) for a, b in zip(old, new))
        # lengths in, lengths and offsets out, slot and position of a token, a page read and written where it moves
        return dict(bytes=4.0 * (4 * case["rows"] + 2 * tokens + 2 * moved), flops=0.0)
    if kind == "logprobs":
        n = case["rows"] * case["vocab"]
        return dict(bytes=float(n * SIZE[case["dtype"]] + case["rows"] * (12 + 8 * case["top"])), flops=6.0 * n)
    d, h, t = case["head_dim"], case["kv_heads"], SIZE[case["dtype"]]
    if kind == "append":
        pages = sum((a + n - 1) // case["page"] - a // case["page"] + 1 for a, n in _runs(case))
        n = case["tokens"] * h * d
        return dict(bytes=float(2 * n * (t + 1) + 16 * pages * h + 4 * case["tokens"]), flops=4.0 * n)
    q = case["heads"] * d
    if kind == "attn":
        lens = _lens(case, case["rows"], case["max_len"])
        seen = [min(n, case["window"]) if case["window"] else n for n in lens]
        pages = sum(-(-n // case["page"]) for n in seen)
        return dict(bytes=float(2 * h * d * sum(seen) + (8 * h + 4) * pages + 2 * len(lens) * q * t),
                    flops=4.0 * q * sum(seen))
    lens = _lens(case, case["seqs"], case["max_len"])
    w = case["window"]
    pairs = sum(n * (n + 1) // 2 if not w or n <= w else w * (w + 1) // 2 + (n - w) * w for n in lens)
    return dict(bytes=float(sum(lens) * (2 * q + 2 * h * d) * t), flops=4.0 * q * pairs)


# ---- the definitions in 64 bits ----

def _nearest(x, kv):
    """The nearest code's value, ties to even."""
    if kv == "i8":
        x = torch.where(torch.isnan(x), torch.zeros_like(x), x)
        return x.clamp(-127, 127).round()
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -20))).clamp(min=-6) - 3)
    return torch.where(torch.isfinite(x), (x / step).round() * step, torch.full_like(x, float("nan")))


def _exact_append(st, x, codes, scale, is_v):
    c = st["case"]
    s, d, h, kv = c["page"], c["head_dim"], c["kv_heads"], c["kv"]
    most = 448.0 if kv == "e4m3" else 127.0
    codes, scale = codes.double(), scale.double()
    by_page = {}
    for i, slot in enumerate(st["slots"].tolist()):
        by_page.setdefault(slot // s, []).append((slot % s, i))
    token = torch.arange(s, device="cuda")[:, None]
    dim = torch.arange(d, device="cuda")[None]
    place = token * d + dim
    if is_v:
        place = ((((token // 16) * 16 + dim % 16) * 4 + (token % 16) // 4) * (d // 16) + dim // 16) * 4 + token % 4
    for page, got in by_page.items():
        offs = torch.tensor([o for o, _ in got], device="cuda")
        rows = x[torch.tensor([i for _, i in got], device="cuda")].double().view(-1, h, d).transpose(0, 1)
        amax = torch.where(torch.isfinite(rows), rows, torch.zeros_like(rows)).abs().amax((1, 2))
        need = torch.exp2(torch.ceil(torch.log2(amax.clamp(min=1e-300) / most)).clamp(E_MIN, E_MAX))
        held = codes[page][:, place]                       # [h, s, d]
        if bool((offs == 0).any()):
            to = need
        else:
            to = torch.maximum(scale[page], need)
            held = torch.where((to > scale[page])[:, None, None], _nearest(held * (scale[page] / to)[:, None, None], kv), held)
        held[:, offs] = _nearest(rows / to[:, None, None], kv)
        codes[page, :, place.reshape(-1)] = held.reshape(h, -1)
        scale[page] = to
    return codes, scale


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "map":
        return None
    if kind == "append":
        kc, ks = _exact_append(st, st["k"], st["k_codes"], st["k_scale"], False)
        vc, vs = _exact_append(st, st["v"], st["v_codes"], st["v_scale"], True)
        return dict(k=kc, k_scale=ks, v=vc, v_scale=vs)
    if kind == "logprobs":
        lp, ent, top = [], [], []
        for x, tok in zip(st["logits"].split(16), st["tokens"].split(16)):
            x = x.double()
            logp = x - torch.logsumexp(x, 1, keepdim=True)
            lp.append(logp.gather(1, tok.long()[:, None])[:, 0])
            ent.append(-torch.where(logp > -INF, logp * torch.exp(logp), torch.zeros_like(logp)).sum(1))
            top.append(torch.topk(logp, case["top"], 1).values)
        return dict(logprob=torch.cat(lp), entropy=torch.cat(ent), top_ids=None, top_logprobs=torch.cat(top))
    d, h, w = case["head_dim"], case["kv_heads"], case["window"]
    g = case["heads"] // h
    if kind == "attn":
        s = case["page"]
        out = torch.zeros(case["rows"], h, g, d, dtype=torch.float64, device="cuda")
        token = torch.arange(s, device="cuda")[:, None]
        dim = torch.arange(d, device="cuda")[None]
        v_at = ((((token // 16) * 16 + dim % 16) * 4 + (token % 16) // 4) * (d // 16) + dim // 16) * 4 + token % 4
        for r, n in enumerate(_lens(case, case["rows"], case["max_len"])):
            if n == 0:
                continue
            first = max(0, n - w) if w else 0
            ids = st["table"][r, :-(-n // s)].long()
            k = (st["k_codes"][ids].double() * st["k_scale"][ids].double()[..., None]).view(-1, h, s, d)
            v = (st["v_codes"][ids].double() * st["v_scale"][ids].double()[..., None])[:, :, v_at]
            k, v = (y.transpose(0, 1).reshape(h, -1, d)[:, first:n] for y in (k, v))
            p = torch.softmax(st["q"][r].double().view(h, g, d) @ k.transpose(1, 2).contiguous() / math.sqrt(d), -1)
            out[r] = p @ v
        return out.view(case["rows"], -1)
    out = torch.empty(st["tokens"], h, g, d, dtype=torch.float64, device="cuda")
    cu = st["cu"].tolist()
    for a, b in zip(cu[:-1], cu[1:]):
        for head in range(h):
            k, v = (st[y][a:b].view(b - a, h, d)[:, head].double() for y in "kv")
            for at in range(a, b, 1024):
                to = min(b, at + 1024)
                q = st["q"][at:to].view(to - at, h, g, d)[:, head].double().transpose(0, 1).contiguous()
                i, j = torch.arange(at - a, to - a, device="cuda")[:, None], torch.arange(b - a, device="cuda")[None]
                gone = (j > i) | (j <= i - w) if w else j > i
                sc = (q @ k.t().contiguous() / math.sqrt(d)).masked_fill(gone, -INF)
                out[at:to, head] = (torch.softmax(sc, -1) @ v).transpose(0, 1)
    return out.view(st["tokens"], -1)
