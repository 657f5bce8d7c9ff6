"""Causal attention of packed prompts and log probabilities on the GPU,
against float64; the serving operators in a run, in a graph, on a stream."""
import numpy as np
import pytest
import torch

import vkv
from gpu_util import dev, stream_ptr
from serve_util import TORCH, Map, Pool, as64, attend, attend_tolerance, half_step, rows_on_device

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.as_tensor(np.asarray(x, dtype=np.int32)).to(dev())


def causal(n, window):
    i, j = np.arange(n)[:, None], np.arange(n)[None]
    return (j <= i) & ((j > i - window) if window else True)


def call(q, k, v, cu, H, Hk, D, dtype, window=0, scale=None, tokens=None, out=None, **kw):
    tokens = q.shape[0] if tokens is None else tokens
    out = torch.full((tokens, H * D), 7.0, dtype=TORCH[dtype], device=dev()) if out is None else out
    need = vkv.prompt_attn_workspace(dtype, len(cu) - 1, tokens, Hk, D)
    ws = torch.full((need + 256,), 0xff, dtype=torch.uint8, device=dev())
    c = i32(cu)
    vkv.prompt_attn(dtype, q.data_ptr(), k.data_ptr(), v.data_ptr(), c.data_ptr(), len(cu) - 1, tokens, H, Hk, D,
                    1 / np.sqrt(D) if scale is None else scale, window, out.data_ptr(), ws.data_ptr(), need,
                    hip_stream=stream_ptr(), **kw)
    assert (ws[need:] == 0xff).all()
    return out


def check(lens, H, Hk, D, dtype, window=0, seed=0, gain=1.0, scale=None, behind=3, v_gain=None):
    rng = np.random.default_rng(seed + sum(lens))
    cu = np.concatenate([[0], np.cumsum(lens)])
    n = int(cu[-1]) + behind
    q, k, v = (rng.standard_normal((n, h * D)) for h in (H, Hk, Hk))
    q *= gain
    if v_gain is not None:
        v *= v_gain(np.arange(n))[:, None]
    q, k, v = (rows_on_device(x, dtype) for x in (q, k, v))
    got = as64(call(q, k, v, cu, H, Hk, D, dtype, window, scale))
    assert (got[cu[-1]:] == 7.0).all()          # rows behind the last prompt stay as they were
    q, k, v = (as64(x).reshape(n, h, D) for x, h in ((q, H), (k, Hk), (v, Hk)))
    worst = 0.0
    for a, b in zip(cu[:-1], cu[1:]):
        if a == b:
            continue
        sc = 1 / np.sqrt(D) if scale is None else scale
        want, mass, vmass = attend(q[a:b], k[a:b], v[a:b], causal(b - a, window), sc)
        p_step = 0.0 if dtype == vkv.F32 else half_step(dtype)
        tol = attend_tolerance(mass, vmass, want, dtype, D, b - a, np.abs(v[a:b]).max(), p_step)
        err = np.abs(got[a:b].reshape(want.shape) - want)
        worst = max(worst, float((err / tol).max()))
        assert (err <= tol).all(), (a, b, err.max(), float((err / tol).max()))
    return worst


@pytest.mark.parametrize("dtype", [vkv.F32, vkv.F16, vkv.BF16])
@pytest.mark.parametrize("H,Hk,D", [(8, 2, 128), (4, 4, 64), (9, 3, 64), (16, 1, 128), (10, 2, 64)])
def test_prompt_attn_ragged(H, Hk, D, dtype):
    check([1, 0, 2, 63, 64, 65, 0, 0, 127, 128, 129, 31, 38], H, Hk, D, dtype)


@pytest.mark.parametrize("dtype", [vkv.F32, vkv.BF16])
@pytest.mark.parametrize("lens", [[1], [38], [256], [257], [700], [0], [0, 0, 5], [300, 1, 1, 1, 450]])
def test_prompt_attn_lengths(lens, dtype):
    check(lens, 8, 2, 128, dtype, behind=0)


@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 100, 500])
@pytest.mark.parametrize("dtype", [vkv.F32, vkv.F16])
def test_prompt_attn_window(window, dtype):
    check([150, 1, 333, 64], 4, 2, 64, dtype, window)


def test_prompt_attn_many_prompts():
    rng = np.random.default_rng(2)
    check(list(rng.integers(0, 9, 300)), 4, 1, 64, vkv.F32)
    check([1] * 70 + [130] + [0] * 64 + [3], 2, 2, 64, vkv.F16)


@pytest.mark.parametrize("n", [63, 64, 65])
def test_prompt_attn_of_about_64_prompts(n):
    """the search for a tile's prompt takes one step up to 64 prompts, then two"""
    rng = np.random.default_rng(n)
    lens = list(rng.integers(0, 20, n))
    lens[3], lens[n // 2], lens[-1] = 200, 333, 131
    check(lens, 4, 1, 64, vkv.BF16)


@pytest.mark.parametrize("window", [0, 2100])
def test_prompt_attn_of_more_than_64_tiles(window):
    check([9, 2300], 1, 1, 128, vkv.F32, window)


def test_prompt_attn_offsets_that_count_rows_many_times():
    """64 prompts that each claim every row: the accesses stay in the arrays, the call ends"""
    rng = np.random.default_rng(11)
    H, Hk, D, n = 2, 1, 64, 300
    q, k, v = (rows_on_device(rng.standard_normal((n, h * D)), vkv.F16) for h in (H, Hk, Hk))
    call(q, k, v, [0, n] * 32 + [0], H, Hk, D, vkv.F16)
    torch.cuda.synchronize()
    want = call(q, k, v, [0, n], H, Hk, D, vkv.F16)
    assert torch.equal(call(q, k, v, [0] * 64 + [n], H, Hk, D, vkv.F16), want)


@pytest.mark.parametrize("gain,scale", [(300.0, None), (1e-30, None), (1.0, -0.1), (1.0, 0.0), (1e30, 1e-31)])
def test_prompt_attn_of_scores_far_apart(gain, scale):
    check([130, 70], 4, 2, 128, vkv.F32, gain=gain, scale=scale)


@pytest.mark.parametrize("dtype", [vkv.F32, vkv.F16, vkv.BF16])
@pytest.mark.parametrize("scale", [1e6, -1e8, 1e20])
def test_prompt_attn_of_scores_beyond_their_own_steps(dtype, scale):
    """scores so large that neighbouring f32 values are several units apart: a row takes its largest key alone (no two
    of these keys are nearly as large), and equal keys share it"""
    rng = np.random.default_rng(14)
    n, D = 150, 64
    q = np.ones((n, D))
    size = rng.permutation(n)               # q . k = 64 * size: exact in every type
    k = np.repeat(size[:, None], D, 1).astype(float)
    k[100:110] = k[99] + 1000
    v = rng.integers(-8, 9, (n, D)).astype(float)
    got = as64(call(*(rows_on_device(x, dtype) for x in (q, k, v)), [0, n], 1, 1, D, dtype, scale=scale))
    for t in range(n):
        s = np.sign(scale) * k[:t + 1, 0]
        want = v[:t + 1][s == s.max()].mean(0)
        assert np.abs(got[t] - want).max() <= 8 * 2 * half_step(dtype) + 1e-6


def test_prompt_attn_values_of_very_different_sizes():
    """by prompt, and by tile of a prompt: f32 rows are scaled by tile"""
    check([200, 100, 150], 4, 2, 64, vkv.F32, v_gain=lambda t: np.where(t < 200, 1e-12, np.where(t < 300, 1e9, 1.0)))
    check([300], 4, 2, 64, vkv.F32, window=40, v_gain=lambda t: 10.0 ** (t // 64 * 3 - 6))
    check([300], 4, 2, 64, vkv.F32, window=40, v_gain=lambda t: 10.0 ** (6 - t // 64 * 3))


@pytest.mark.parametrize("dtype", [vkv.F32, vkv.F16, vkv.BF16])
@pytest.mark.parametrize("window", [0, 30])
def test_prompt_attn_keys_out_of_sight_do_nothing(dtype, window):
    """NaN and infinities in a later token, or before the window, reach no row that does not attend to them; the rows
    that do get them"""
    rng = np.random.default_rng(6)
    H, Hk, D, n = 4, 2, 64, 150
    q, k, v = (rng.standard_normal((n, h * D)) for h in (H, Hk, Hk))
    clean = as64(call(*(rows_on_device(x, dtype) for x in (q, k, v)), [0, n], H, Hk, D, dtype, window))
    v[70, 5], v[70, D + 6], v[71, 7], v[90, 5] = np.inf, np.nan, -np.inf, -np.inf
    k[100, 3] = np.nan
    got = as64(call(*(rows_on_device(x, dtype) for x in (q, k, v)), [0, n], H, Hk, D, dtype, window))
    got, clean = got.reshape(n, H, D), clean.reshape(n, H, D)
    t = np.arange(n)
    sees = lambda key: (t >= key) & ((t < key + window) if window else True)  # noqa: E731
    want = clean.copy()
    want[sees(70), :2, 5] = np.inf
    want[sees(90) & ~sees(70), :2, 5] = -np.inf
    want[sees(90) & sees(70), :2, 5] = np.nan
    want[sees(70), 2:, 6] = np.nan
    want[sees(71), :2, 7] = -np.inf
    want[sees(100), :2] = np.nan
    same = (got == want) | (np.isnan(got) & np.isnan(want))
    # the other dims of those rows are computed as before
    assert same.all(), np.argwhere(~same)[:5].tolist()


def test_prompt_attn_rows_of_one_wide_array():
    """q, k and v as one product leaves them, out into another wide array"""
    rng = np.random.default_rng(9)
    H, Hk, D, n = 6, 2, 64, 100
    width = (H + 2 * Hk) * D + 64
    qkv = rows_on_device(rng.standard_normal((n, width)), vkv.BF16)
    q, k, v = qkv, qkv[:, H * D:], qkv[:, (H + Hk) * D:]
    out = torch.full((n, 2 * H * D), 7.0, dtype=torch.bfloat16, device=dev())
    call(q, k, v, [0, 60, n], H, Hk, D, vkv.BF16, out=out, tokens=n, q_stride=width, k_stride=width, v_stride=width,
         out_stride=2 * H * D)
    packed = [x[:, :w].contiguous() for x, w in ((q, H * D), (k, Hk * D), (v, Hk * D))]
    want = call(*packed, [0, 60, n], H, Hk, D, vkv.BF16)
    assert torch.equal(out[:, :H * D], want) and (out[:, H * D:] == 7.0).all()


def test_prompt_attn_offsets_outside_the_rows_are_held_to_them():
    """offsets that are none: every access stays in the arrays, rows of prompts that are well given are right"""
    rng = np.random.default_rng(10)
    H, Hk, D, n = 4, 2, 64, 200
    q, k, v = (rows_on_device(rng.standard_normal((n, h * D)), vkv.F32) for h in (H, Hk, Hk))
    want = call(q, k, v, [0, 90, 200], H, Hk, D, vkv.F32)
    got = call(q, k, v, [0, 90, 2 ** 31 - 1], H, Hk, D, vkv.F32)
    assert torch.equal(got, want)
    got = call(q, k, v, [-5, 90, 40, 200], H, Hk, D, vkv.F32)
    assert torch.equal(got[:40], want[:40])     # rows [40, 90) are two prompts'
    got = call(q, k, v, [200, 200], H, Hk, D, vkv.F32)
    assert (got == 7.0).all()
    got = call(q, k, v, [90, 200], H, Hk, D, vkv.F32)
    assert torch.equal(got[90:], want[90:]) and (got[:90] == 7.0).all()


@pytest.fixture
def many_groups(monkeypatch):
    """200 empty prompts behind the others: the form for many work groups takes what the other form took above"""
    real = call

    def padded(q, k, v, cu, *rest, **kw):
        return real(q, k, v, list(cu) + [cu[-1]] * 200, *rest, **kw)
    monkeypatch.setitem(globals(), "call", padded)


@pytest.mark.parametrize("dtype", [vkv.F32, vkv.F16, vkv.BF16])
@pytest.mark.parametrize("H,Hk,D", [(8, 2, 128), (4, 4, 64), (9, 3, 64), (16, 1, 128)])
def test_prompt_attn_many_groups_ragged(H, Hk, D, dtype, many_groups):
    check([1, 0, 2, 63, 64, 65, 0, 0, 127, 128, 129, 31, 38, 300], H, Hk, D, dtype)


@pytest.mark.parametrize("window", [1, 31, 64, 65, 100, 500])
@pytest.mark.parametrize("dtype,D", [(vkv.F32, 128), (vkv.F32, 64), (vkv.F16, 64)])
def test_prompt_attn_many_groups_window(window, dtype, D, many_groups):
    check([150, 1, 333, 64], 4, 2, D, dtype, window)


@pytest.mark.parametrize("dtype", [vkv.F32, vkv.F16, vkv.BF16])
def test_prompt_attn_many_groups_of_every_kind(dtype, many_groups):
    for window in (0, 30):
        test_prompt_attn_keys_out_of_sight_do_nothing(dtype, window)
    for scale in (1e6, -1e8, 1e20):
        test_prompt_attn_of_scores_beyond_their_own_steps(dtype, scale)
    if dtype == vkv.F32:
        for gain, scale in ((300.0, None), (1e-30, None), (1.0, -0.1), (1.0, 0.0), (1e30, 1e-31)):
            test_prompt_attn_of_scores_far_apart(gain, scale)
        test_prompt_attn_values_of_very_different_sizes()
        test_prompt_attn_offsets_outside_the_rows_are_held_to_them()
        test_prompt_attn_of_more_than_64_tiles(0)
    test_prompt_attn_rows_of_one_wide_array()


@pytest.mark.parametrize("dtype", [vkv.F32, vkv.F16, vkv.BF16])
@pytest.mark.parametrize("D,n", [(64, 4300), (128, 2200)])
def test_prompt_attn_of_few_rows_and_many_tiles(dtype, D, n):
    """more than 64 tiles of keys, four waves on them; one query head, so that the rows are few"""
    check([n], 1, 1, D, dtype, window=n - 100)


# ---- log probabilities ----
def logprobs(x, tokens, top, dtype, row_stride=0, vocab=None, rows=None):
    n, v = x.shape[0] if rows is None else rows, x.shape[1] if vocab is None else vocab
    lp, ent = torch.full((n + 1,), 7.0, device=dev()), torch.full((n + 1,), 7.0, device=dev())
    ids = torch.full((n + 1, top), -9, dtype=torch.int32, device=dev())
    tlp = torch.full((n + 1, top), 7.0, device=dev())
    need = vkv.logprobs_workspace(n, v, top)
    ws = torch.full((need + 64,), 0xff, dtype=torch.uint8, device=dev())
    t = i32(tokens)
    vkv.logprobs(dtype, x.data_ptr(), n, v, t.data_ptr(), lp.data_ptr(), ent.data_ptr(), top, ids.data_ptr(),
                 tlp.data_ptr(), ws.data_ptr(), need, row_stride=row_stride, hip_stream=stream_ptr())
    assert (ws[need:] == 0xff).all() and lp[n] == 7 and ent[n] == 7 and (ids[n] == -9).all()
    return as64(lp[:n]), as64(ent[:n]), ids[:n].cpu().numpy(), as64(tlp[:n])


def logprobs_reference(x, tokens, top):
    m = x.max(1, keepdims=True)
    with np.errstate(all="ignore"):
        logp = x - m - np.log(np.exp(x - m).sum(1, keepdims=True))
        ent = -np.where(logp > -np.inf, np.exp(logp) * logp, 0.0).sum(1)
    ids = np.argsort(-x, axis=1, kind="stable")[:, :top]
    return logp[np.arange(len(x)), tokens], ent, ids, np.take_along_axis(logp, ids, 1)


def check_logprobs(x, tokens, top, dtype, **kw):
    """A term exp(x - m) is off by |x - m| 2^-24 (its argument) and 2 2^-24, but terms of |x - m| > 20 weigh nothing;
    sums of n terms in trees over chunks by (32 + log2 n) 2^-24 at the most; the results' own rounding."""
    got = logprobs(rows_on_device(x, dtype), tokens, top, dtype, **kw)
    x = as64(rows_on_device(x, dtype))
    want = logprobs_reference(x, tokens, top)
    rel = (24 + 32 + np.log2(x.shape[1])) * 2.0 ** -24
    lp_tol = rel + 3 * 2.0 ** -24 * np.abs(want[0]) + 1e-30
    assert np.array_equal(got[2], want[2])
    assert (np.abs(got[0] - want[0]) <= lp_tol).all(), np.abs(got[0] - want[0]).max()
    assert (np.abs(got[3] - want[3]) <= rel + 3 * 2.0 ** -24 * np.abs(want[3])).all()
    # the entropy adds the terms (x - m) exp(x - m), whose mean is at most log n + the entropy
    ent_tol = rel * (2 + 2 * np.log(x.shape[1]))
    assert (np.abs(got[1] - want[1]) <= ent_tol).all(), (np.abs(got[1] - want[1]).max(), ent_tol)


@pytest.mark.parametrize("dtype", [vkv.F32, vkv.F16, vkv.BF16])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 2, 2), (2, 7, 7), (5, 33, 32), (4, 1000, 0), (2, 2049, 1),
                                            (3, 8191, 5), (2, 8193, 32), (1, 131072, 20), (70, 32003, 10)])
def test_logprobs(rows, vocab, top, dtype):
    rng = np.random.default_rng(rows + vocab)
    x = rng.standard_normal((rows, vocab)) * 4
    check_logprobs(x, rng.integers(0, vocab, rows), top, dtype)


def test_logprobs_of_many_rows_take_the_larger_chunks():
    rng = np.random.default_rng(1)
    for dtype in (vkv.F32, vkv.BF16):
        check_logprobs(rng.standard_normal((300, 20001)) * 3, rng.integers(0, 20001, 300), 32, dtype)


@pytest.mark.parametrize("dtype", [vkv.F32, vkv.F16])
def test_logprobs_ties_go_to_the_lowest_id(dtype):
    rng = np.random.default_rng(3)
    n = 20000
    for x in (np.zeros((2, n)), rng.integers(0, 2, (2, n)).astype(float), rng.integers(-3, 4, (2, n)) * 0.5,
              np.tile(np.arange(n) % 40 / 4, (2, 1)), np.sort(rng.standard_normal((2, n)), 1),
              -np.sort(rng.standard_normal((2, n)), 1), np.where(rng.random((2, n)) < 0.5, 0.0, -0.0)):
        check_logprobs(x, [0, n - 1], 32, dtype)


@pytest.mark.parametrize("dtype", [vkv.F32, vkv.BF16])
def test_logprobs_of_many_rows_of_every_kind(dtype):
    """several pieces to a work group: values that rise, so that the first piece's limit keeps nothing out, or fall;
    many equal ones; few that are not -inf, in the first piece or behind it; NaN and +inf"""
    rng = np.random.default_rng(12)
    n, v, top = 200, 40001, 32
    x = rng.standard_normal((n, v)) * 3
    x[:20] = np.sort(x[:20], 1)
    x[20:40] = -np.sort(-x[20:40], 1)
    x[40:60] = rng.integers(0, 3, (20, v))
    for r in range(60, 80):
        x[r, rng.permutation(v)[:v - 1 - r % 40]] = -np.inf
    x[80:85, :39990] = -np.inf
    x[85:90, 11:] = -np.inf
    x[90:95] = -np.inf
    x[95:100, 0] = 1e6 if dtype == vkv.F32 else 1e4
    tokens = rng.integers(0, v, n)
    x[100, 39999], x[101, 3], x[102, 20000] = np.nan, np.inf, np.nan
    got = logprobs(rows_on_device(x, dtype), tokens, top, dtype)
    x = as64(rows_on_device(x, dtype))
    rows = np.r_[0:90, 95:100, 103:n]
    want = logprobs_reference(x[rows], tokens[rows], top)
    assert np.array_equal(got[2][rows], want[2])
    rel = (24 + 32 + np.log2(v)) * 2.0 ** -24
    with np.errstate(invalid="ignore"):
        for g, w in ((got[0][rows], want[0]), (got[3][rows], want[3])):
            assert ((np.abs(g - w) <= rel + 3 * 2.0 ** -24 * np.abs(w)) | (g == w)).all()
    assert (np.abs(got[1][rows] - want[1]) <= rel * (2 + 2 * np.log(v))).all()
    for r in range(90, 95):
        assert got[0][r] == -np.inf and got[1][r] == 0 and got[2][r].tolist() == list(range(top)) and (got[3][r] == -np.inf).all()
    for r, first in ((100, 39999), (101, 3), (102, 20000)):
        assert np.isnan(got[0][r]) and np.isnan(got[1][r]) and np.isnan(got[3][r]).all() and got[2][r, 0] == first


@pytest.mark.parametrize("dtype", [vkv.F32, vkv.F16])
@pytest.mark.parametrize("vocab,rows", [(7, 3), (5000, 5), (20001, 300)])
def test_logprobs_of_rows_that_are_sure(vocab, rows, dtype):
    """a probability next to 1: its logarithm and the entropy to f32's relative precision.  The other terms' sum has
    terms off by |x - m| 2^-24 (their arguments, below 40 here) and 2 2^-24, and is one in trees as above; the logarithm
    and the division add 3 2^-24; the entropy's terms are these and their products with |x - m|, all of one sign"""
    rng = np.random.default_rng(15)
    x = rng.uniform(-3, 3, (rows, vocab))
    token = rng.integers(0, vocab, rows)
    x[np.arange(rows), token] = np.arange(rows) % 20 + 12
    dev_x = rows_on_device(x, dtype)
    got = logprobs(dev_x, token, 1, dtype)
    x = as64(dev_x)
    d = x - x[np.arange(rows), token][:, None]
    e = np.exp(d)
    e[np.arange(rows), token] = 0
    rest = e.sum(1)
    lp = -np.log1p(rest)
    ent = np.log1p(rest) - (e * d).sum(1) / (1 + rest)
    rel = (40 + 2 + 32 + np.log2(vocab) + 3) * 2.0 ** -24
    assert (np.abs(got[0] - lp) <= rel * np.abs(lp)).all() and np.array_equal(got[0], got[3][:, 0])
    assert (np.abs(got[1] - ent) <= 2 * rel * ent).all()


@pytest.mark.parametrize("vocab,rows", [(5000, 5), (20001, 300)])
def test_logprobs_of_large_logits(vocab, rows):
    """spread over, or all near, magnitudes at which a unit is many, few and none of f32's steps"""
    rng = np.random.default_rng(13)
    x = rng.standard_normal((rows, vocab)) * np.array([1e2, 1e4, 1e6, 1e9, 1e30])[np.arange(rows) % 5, None]
    check_logprobs(x, rng.integers(0, vocab, rows), 3, vkv.F32)
    x = rng.standard_normal((rows, vocab)) + np.array([1e2, -1e4, 1e6, -3e7, 1e10])[np.arange(rows) % 5, None]
    check_logprobs(x, rng.integers(0, vocab, rows), 3, vkv.F32)


@pytest.mark.parametrize("dtype", [vkv.F32, vkv.F16])
@pytest.mark.parametrize("vocab,rows", [(999, 12), (30001, 12), (30001, 250)])
def test_logprobs_of_rows_of_equal_values(vocab, rows, dtype):
    """masks of the type's lowest value with a few logits left, more or fewer than are asked for; rows of one value; two
    values; equal values in many places and pieces"""
    rng = np.random.default_rng(16)
    low = float(torch.finfo(TORCH[dtype]).min)
    x = np.full((rows, vocab), low)
    for r in range(rows):
        kind = r % 6
        some = rng.permutation(vocab)[:[3, 32, 200, 0, 40, 17][kind]]
        if kind < 3:
            x[r, some] = rng.standard_normal(len(some))
        else:
            x[r] = 0.0
            x[r, some] = 1.0 if kind == 4 else rng.integers(0, 3, len(some))
    check_logprobs(x, rng.integers(0, vocab, rows), 32, dtype)
    check_logprobs(x, rng.integers(0, vocab, rows), 5, dtype)


def test_logprobs_masked_rows():
    """-inf has no probability; a row of it alone has no distribution; NaN and +inf make a row NaN"""
    rng = np.random.default_rng(4)
    n = 9000
    x = rng.standard_normal((6, n))
    x[0, rng.permutation(n)[:n - 3]] = -np.inf
    x[1] = -np.inf
    x[2, 17] = np.nan
    x[3, 18] = np.inf
    x[4, 1:] = -np.inf
    x[5] = -np.finfo(np.float32).max
    fine = np.flatnonzero(np.isfinite(x[0]))
    token = int(fine[0])
    lp, ent, ids, tlp = logprobs(rows_on_device(x, vkv.F32), [token, 5, 3, 3, 0, 8999], 8, vkv.F32)
    for r in (0, 4, 5):
        wl, we, wi, wt = logprobs_reference(x[[r]].astype(np.float32).astype(np.float64), [[token], 0, 0, 0, [0], [8999]][r], 8)
        assert np.array_equal(ids[r], wi[0])
        assert np.allclose(lp[r], wl, atol=1e-5) and np.allclose(ent[r], we, atol=1e-4)
        assert np.allclose(tlp[r][np.isfinite(wt[0])], wt[0][np.isfinite(wt[0])], atol=1e-5)
        assert np.array_equal(np.isfinite(tlp[r]), np.isfinite(wt[0]))
    assert lp[1] == -np.inf and ent[1] == 0 and ids[1].tolist() == list(range(8)) and (tlp[1] == -np.inf).all()
    for r, first in ((2, 17), (3, 18)):
        assert np.isnan(lp[r]) and np.isnan(ent[r]) and np.isnan(tlp[r]).all() and ids[r, 0] == first


def test_logprobs_tokens_that_are_none():
    x = rows_on_device(np.zeros((4, 10)), vkv.F32)
    lp = logprobs(x, [-1, 10, -2, 9], 1, vkv.F32)[0]
    assert lp[0] == 0 and np.isnan(lp[1]) and np.isnan(lp[2]) and abs(lp[3] + np.log(10)) < 1e-6


@pytest.mark.parametrize("dtype", [vkv.F32, vkv.BF16])
@pytest.mark.parametrize("stride", [0, 1, 3, 8])
def test_logprobs_rows_at_any_place(dtype, stride):
    """odd row lengths and strides: rows begin anywhere; their neighbours are not read into them"""
    rng = np.random.default_rng(5)
    n, v = 5, 4999
    x = rng.standard_normal((n, v))
    wide = np.full((n, v + stride), 1e4)
    wide[:, :v] = x
    tokens = rng.integers(0, v, n)
    a = logprobs(rows_on_device(wide, dtype), tokens, 9, dtype, row_stride=v + stride, vocab=v)
    want = logprobs_reference(as64(rows_on_device(x, dtype)), tokens, 9)
    assert np.array_equal(a[2], want[2]) and np.allclose(a[0], want[0], atol=1e-5) and np.allclose(a[1], want[1], atol=1e-4)


def test_logprobs_parts_may_be_left_out():
    x = rows_on_device(np.arange(100.0)[None] / 10, vkv.F32)
    ent = torch.zeros(1, device=dev())
    ws = torch.empty(vkv.logprobs_workspace(1, 100, 0), dtype=torch.uint8, device=dev())
    vkv.logprobs(vkv.F32, x.data_ptr(), 1, 100, 0, 0, ent.data_ptr(), 0, 0, 0, ws.data_ptr(), ws.numel(), hip_stream=stream_ptr())
    want = logprobs_reference(as64(x), [0], 1)[1]
    assert abs(ent.item() - want[0]) < 1e-4
    ids, lps = torch.zeros(1, 1, dtype=torch.int32, device=dev()), torch.zeros(1, 1, device=dev())
    ws = torch.empty(vkv.logprobs_workspace(1, 100, 1), dtype=torch.uint8, device=dev())
    vkv.logprobs(vkv.F32, x.data_ptr(), 1, 100, 0, 0, 0, 1, ids.data_ptr(), lps.data_ptr(), ws.data_ptr(), ws.numel(),
                 hip_stream=stream_ptr())
    assert ids.item() == 99


# ---- together ----
class Server:
    """What a program keeps to answer requests from one pool: every buffer of a step at fixed addresses."""

    def __init__(self, n_req, page, stride, n_pages, H, Hk, D, vocab, code, dtype, max_tokens, seed):
        self.H, self.Hk, self.D, self.vocab, self.dtype, self.n_req = H, Hk, D, vocab, dtype, n_req
        self.max_len = stride * page
        self.map = Map(page, n_pages, n_req, stride)
        self.map.room(max_tokens)
        self.pool = Pool(code, n_pages, page, Hk, D)
        g = torch.Generator(device=dev()).manual_seed(seed)
        t = TORCH[dtype]
        self.k, self.v = (torch.randn(max_tokens, Hk * D, generator=g, device=dev()).to(t) for _ in "kv")
        self.q = torch.randn(max_tokens, H * D, generator=g, device=dev()).to(t)
        self.head = torch.randn(H * D, vocab, generator=g, device=dev()) / 8
        self.out = torch.zeros(max_tokens, H * D, dtype=t, device=dev())
        self.new = torch.zeros(n_req, dtype=torch.int32, device=dev())
        self.logits = torch.zeros(n_req, vocab, device=dev())
        self.tokens = torch.zeros(n_req, dtype=torch.int32, device=dev())
        self.lp, self.ent = torch.zeros(n_req, device=dev()), torch.zeros(n_req, device=dev())
        self.ids = torch.zeros(n_req, 4, dtype=torch.int32, device=dev())
        self.tlp = torch.zeros(n_req, 4, device=dev())
        size = max(vkv.paged_attn_workspace(self.pool.desc, n_req, H, self.max_len),
                   vkv.prompt_attn_workspace(dtype, n_req, max_tokens, Hk, D), vkv.logprobs_workspace(n_req, vocab, 4))
        self.ws = torch.zeros(size, dtype=torch.uint8, device=dev())

    def admit(self):
        """prompts: their rows into the pages, their attention"""
        m = self.map
        m.call(self.new)
        self.pool.append(m.slots, self.k, self.v, self.dtype)
        vkv.prompt_attn(self.dtype, self.q.data_ptr(), self.k.data_ptr(), self.v.data_ptr(), m.cu.data_ptr(), self.n_req,
                        m.max_tokens, self.H, self.Hk, self.D, 0.1, 0, self.out.data_ptr(), self.ws.data_ptr(),
                        self.ws.numel(), hip_stream=stream_ptr())

    def step(self):
        """one token of every request"""
        m = self.map
        m.call(self.new)
        self.pool.append(m.slots, self.k, self.v, self.dtype)
        vkv.paged_attn(self.pool.desc, 0, m.table.data_ptr(), m.stride, m.lens.data_ptr(), self.n_req, self.max_len,
                       self.dtype, self.q.data_ptr(), self.out.data_ptr(), self.H, 0.1, 0, self.ws.data_ptr(),
                       self.ws.numel(), hip_stream=stream_ptr())
        torch.mm(self.out[:self.n_req].float(), self.head, out=self.logits)
        vkv.argmax(self.logits.data_ptr(), self.vocab, self.tokens.data_ptr(), hip_stream=stream_ptr())
        vkv.logprobs(vkv.F32, self.logits.data_ptr(), self.n_req, self.vocab, self.tokens.data_ptr(), self.lp.data_ptr(),
                     self.ent.data_ptr(), 4, self.ids.data_ptr(), self.tlp.data_ptr(), self.ws.data_ptr(),
                     self.ws.numel(), hip_stream=stream_ptr())


def server(seed=5):
    return Server(n_req=4, page=16, stride=8, n_pages=40, H=8, Hk=2, D=64, vocab=999, code=vkv.E4M3, dtype=vkv.F32,
                  max_tokens=120, seed=seed)


def test_a_run_of_the_operators():
    """prompts are admitted, then tokens follow: attention over the pages is the attention over the rows, as far as
    8-bit codes go, and exactly that of the codes; the first alternative is the greedy token"""
    s = server()
    s.new.copy_(i32([33, 1, 0, 70]))
    s.admit()
    torch.cuda.synchronize()
    assert s.map.cu.tolist() == [0, 33, 34, 34, 104] and s.map.status.item() == 0
    k, v, q = (as64(x).reshape(120, -1, 64) for x in (s.k, s.v, s.q))
    got = as64(s.out).reshape(120, 8, 64)
    past = {}
    for r, (a, b) in enumerate([(0, 33), (33, 34), (34, 34), (34, 104)]):
        want, mass, vmass = attend(q[a:b], k[a:b], v[a:b], causal(b - a, 0), 0.1)
        assert (np.abs(got[a:b] - want) <= attend_tolerance(mass, vmass, want, vkv.F32, 64, b - a + 1, 5.0)).all()
        past[r] = (list(k[a:b]), list(v[a:b]))
    lens = [33, 1, 0, 70]
    for n in range(5):
        s.k.add_(0.25)
        s.v.mul_(1.1)
        lens = [x + 1 for x in lens]
        s.new.copy_(i32(lens))
        s.step()
        torch.cuda.synchronize()
        kk, vv, out = as64(s.k).reshape(120, -1, 64), as64(s.v).reshape(120, -1, 64), as64(s.out)[:4].reshape(4, 8, 64)
        (kc, ks), (vc, vs) = s.pool.read()
        table = s.map.table.cpu().numpy()
        for r in range(4):
            past[r][0].append(kk[r])
            past[r][1].append(vv[r])
            ids, off = [table[r, i // 16] for i in range(lens[r])], [i % 16 for i in range(lens[r])]
            pk, pv = ((c[ids, :, off] * sc[ids][..., None]) for c, sc in ((kc, ks), (vc, vs)))
            # codes: half a step is 2^-4 of the value, or of the smallest normal code; a code may have moved to a
            # larger scale once more for each time its page's scale grew
            for code, exact in ((pk, np.array(past[r][0])), (pv, np.array(past[r][1]))):
                assert np.abs(code - exact).max() <= np.abs(exact).max() * 2.0 ** -4 * 1.3
            live = np.ones((1, lens[r]), bool)
            want, mass, vmass = attend(q[r][None], pk, pv, live, 0.1)
            assert (np.abs(out[r] - want[0]) <= attend_tolerance(mass, vmass, want, vkv.F32, 64, lens[r], 9.0)[0]).all()
        assert s.ids[0, 0] == s.tokens[0] and s.lp[0] == s.tlp[0, 0]
    # everybody leaves
    s.new.zero_()
    s.map.call(s.new)
    assert s.map.n_free.item() == 40 and sorted(s.map.free.tolist()) == list(range(40))


def test_a_step_in_a_graph():
    """captured once, replayed with other work between the replays, each against the same steps run eagerly"""
    eager, s = server(7), server(7)
    side = torch.cuda.Stream()
    for x in (eager, s):
        x.new.copy_(i32([20, 3, 40, 1]))
        x.admit()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        s.new.copy_(s.map.lens)
        s.step()            # a step of no new tokens: warms up, changes nothing
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.step()
    lens = [20, 3, 40, 1]
    for n in range(6):
        lens = [x + 1 for x in lens] if n != 3 else [lens[0] + 1, 0, lens[2] - 5, lens[3] + 1]
        for x in (eager, s):
            x.new.copy_(i32(lens))
            x.k.add_(0.125)
            x.q.mul_(1.01)
        eager.step()
        graph.replay()
        torch.cuda.synchronize()
        for name in ("out", "logits", "tokens", "lp", "ent", "ids", "tlp"):
            a, b = getattr(eager, name), getattr(s, name)
            assert torch.equal(a.nan_to_num(), b.nan_to_num()), (n, name)
        for name in ("table", "free", "n_free", "lens", "cu", "slots", "positions", "status"):
            assert torch.equal(getattr(eager.map, name), getattr(s.map, name)), (n, name)
        for a, b in zip(eager.pool.codes + eager.pool.scale, s.pool.codes + s.pool.scale):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_prompts_in_a_graph():
    """admitting prompts, captured once, replayed with other prompts and other work between the replays"""
    eager, s = server(8), server(8)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        s.admit()           # of no prompt: warms up, changes nothing
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.admit()
    for lens in ([20, 3, 40, 1], [0, 0, 0, 120], [128, 0, 0, 0], [1, 1, 1, 1], [64, 0, 56, 0]):
        for x in (eager, s):
            x.out.fill_(7.0)
            x.new.zero_()
            x.map.call(x.new)           # all pages back
            x.new.copy_(i32(lens))
            x.v.add_(0.5)
        eager.admit()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(eager.out, s.out) and eager.map.status.item() == (2 if sum(lens) > 120 else 0)
        used = sum(lens) if sum(lens) <= 120 else 0
        assert (s.out[used:] == 7.0).all() and not (used and (s.out[:used] == 7.0).all())
        for a, b in zip(eager.pool.codes + eager.pool.scale, s.pool.codes + s.pool.scale):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_a_step_on_another_stream():
    """two servers on two streams at once, with workspaces of their own, against one after the other"""
    alone = [server(1), server(2)]
    both = [server(1), server(2)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()

    def life(s):
        lens = [17, 60, 2, 9]
        s.new.copy_(torch.tensor(lens, dtype=torch.int32), non_blocking=False)
        s.admit()
        for _ in range(10):
            s.new.add_(1)
            s.step()

    for s in alone:
        life(s)
        torch.cuda.synchronize()
    for s, st in zip(both, streams):
        with torch.cuda.stream(st):
            life(s)
    torch.cuda.synchronize()
    for a, b in zip(alone, both):
        for name in ("out", "logits", "lp", "ent", "ids", "tlp"):
            assert torch.equal(getattr(a, name), getattr(b, name)), name


def test_the_same_call_twice_gives_the_same_bits():
    rng = np.random.default_rng(20)
    q, k, v = (rows_on_device(rng.standard_normal((700, h * 128)), vkv.F32) for h in (8, 2, 2))
    a, b = (call(q, k, v, [0, 300, 700], 8, 2, 128, vkv.F32) for _ in range(2))
    assert torch.equal(a, b)
    x = rows_on_device(rng.standard_normal((3, 50000)), vkv.F32)
    a, b = (logprobs(x, [1, 2, 3], 32, vkv.F32) for _ in range(2))
    assert all(np.array_equal(i, j) for i, j in zip(a, b))
