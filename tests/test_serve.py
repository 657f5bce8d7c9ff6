"""Refusals of the batched serving operators, without a GPU: every check is
made before anything is launched, and empty calls do nothing."""
import ctypes

import pytest

import vkv

L = vkv.lib
A = 1 << 20       # an aligned address that no refused call follows


def pages(**kw):
    d = dict(k=A, v=A, k_scale=A, v_scale=A, dtype=vkv.E4M3, n_layers=2, n_pages=10, page_size=16, n_kv_heads=8,
             head_dim=128)
    d.update(kw)
    return vkv.Pages(*[d[f] for f, _ in vkv.Pages._fields_])


def refused(call, status=vkv.INVALID_ARGUMENT, text=None):
    with pytest.raises(vkv.VkvError) as e:
        call()
    assert e.value.status == status, e.value
    if text:
        assert text in e.value.message


MAP = dict(len_old=A, len_new=A, n_req=3, page_size=16, n_pages=10, table=A, table_stride=4, free_pages=A, n_free=A,
           n_free_out=A, max_tokens=8, len_out=A, cu_new=A, slots=A, positions=A, status=A)


@pytest.mark.parametrize("change", [
    dict(n_req=0), dict(n_req=-1), dict(page_size=0), dict(page_size=24), dict(page_size=512), dict(n_pages=0),
    dict(n_pages=1 << 28), dict(table_stride=0), dict(table_stride=1 << 28), dict(max_tokens=-1), dict(len_old=0),
    dict(len_new=0), dict(table=0), dict(free_pages=0), dict(n_free=0), dict(n_free_out=0), dict(len_out=0),
    dict(cu_new=0), dict(slots=0), dict(positions=0), dict(status=0), dict(table=A + 2), dict(slots=A + 1)])
def test_page_map_refuses(change):
    refused(lambda: vkv.page_map(**{**MAP, **change}), text="page map")


POOLS = [dict(dtype=vkv.F16), dict(dtype=vkv.Q8_0), dict(page_size=8), dict(page_size=48), dict(page_size=512),
         dict(head_dim=96), dict(head_dim=256), dict(n_layers=0), dict(n_pages=0), dict(n_kv_heads=0),
         dict(n_pages=1 << 27), dict(n_pages=(1 << 27) - 1, n_kv_heads=17)]
BASES = [dict(k=0), dict(v=0), dict(k_scale=0), dict(v_scale=0), dict(k=A + 8), dict(v_scale=A + 2)]


@pytest.mark.parametrize("pool", POOLS + BASES)
def test_pages_are_checked(pool):
    p = pages(**pool)
    refused(lambda: vkv.pages_append(p, 0, A, 4, vkv.F32, A, A), text="pages append")
    refused(lambda: vkv.paged_attn(p, 0, A, 8, A, 2, 100, vkv.F32, A, A, 32, 0.1, ws=A, ws_bytes=1 << 30),
            text="paged attention")
    if pool in POOLS:
        assert vkv.paged_attn_workspace(p, 2, 32, 100) == 0


APPEND = dict(layer=0, slots=A, n_tokens=4, dtype=vkv.F32, k=A, v=A, row_stride=0)


@pytest.mark.parametrize("change", [
    dict(layer=-1), dict(layer=2), dict(slots=0), dict(slots=A + 2), dict(n_tokens=-1), dict(n_tokens=1 << 24),
    dict(dtype=vkv.Q8_0), dict(dtype=vkv.I8), dict(k=0), dict(v=0), dict(k=A + 4), dict(row_stride=1023),
    dict(row_stride=1026), dict(row_stride=-1024), dict(dtype=vkv.F16, row_stride=1028)])
def test_append_refuses(change):
    refused(lambda: vkv.pages_append(pages(), **{**APPEND, **change}), text="pages append")


ATTN = dict(layer=0, table=A, table_stride=8, lens=A, n_rows=3, max_len=128, dtype=vkv.F32, q=A, out=A, n_q_heads=32,
            scale=0.1, window=0, ws=A, ws_bytes=1 << 30)


@pytest.mark.parametrize("change", [
    dict(layer=-1), dict(layer=2), dict(table=0), dict(lens=0), dict(n_rows=-1), dict(n_rows=1 << 22),
    dict(max_len=-1), dict(max_len=129), dict(table_stride=-1), dict(window=-1), dict(dtype=vkv.Q8_0),
    dict(q=0), dict(out=0), dict(q=A + 4), dict(n_q_heads=30), dict(n_q_heads=4), dict(n_q_heads=0),
    dict(scale=float("nan")), dict(scale=float("inf")), dict(q_stride=4095), dict(q_stride=4098), dict(out_stride=4),
    dict(table_stride=0, max_len=(1 << 31) - 1), dict(table=A + 2)])
def test_paged_attn_refuses(change):
    refused(lambda: vkv.paged_attn(pages(), **{**ATTN, **change}), text="paged attention")


def test_paged_attn_workspace():
    p = pages(n_pages=1000)
    long = {**ATTN, "table_stride": 512, "max_len": 8192}
    need = vkv.paged_attn_workspace(p, 3, 32, 8192)
    assert need > 0
    refused(lambda: vkv.paged_attn(p, **{**long, "ws_bytes": 0}), vkv.BUFFER_TOO_SMALL, "workspace")
    refused(lambda: vkv.paged_attn(p, **{**long, "ws": 0, "ws_bytes": need}), text="workspace")
    refused(lambda: vkv.paged_attn(p, **{**long, "ws": A + 4, "ws_bytes": need}), text="workspace")
    assert vkv.paged_attn_workspace(p, -1, 32, 8192) == 0
    assert vkv.paged_attn_workspace(p, 3, 33, 8192) == 0


PROMPT = dict(dtype=vkv.F32, q=A, k=A, v=A, cu_seqlens=A, n_seq=2, n_tokens=100, n_q_heads=32, n_kv_heads=8,
              head_dim=128, scale=0.1, window=0, out=A, ws=A, ws_bytes=1 << 40)


@pytest.mark.parametrize("change", [
    dict(dtype=vkv.Q8_0), dict(dtype=vkv.E4M3), dict(q=0), dict(k=0), dict(v=0), dict(out=0), dict(cu_seqlens=0),
    dict(cu_seqlens=A + 1), dict(n_seq=-1), dict(n_tokens=-1), dict(n_q_heads=12), dict(n_kv_heads=0),
    dict(n_q_heads=4), dict(head_dim=96), dict(scale=float("nan")), dict(window=-1), dict(q=A + 8), dict(k_stride=1000),
    dict(v_stride=1026), dict(out_stride=-4096), dict(ws=0), dict(ws=A + 16), dict(n_seq=1 << 24),
    dict(n_tokens=(1 << 31) - 1)])
def test_prompt_attn_refuses(change):
    refused(lambda: vkv.prompt_attn(**{**PROMPT, **change}), text="prompt attention")


def test_prompt_attn_workspace():
    need = vkv.prompt_attn_workspace(vkv.F32, 2, 100, 8, 128)
    assert need > 0
    refused(lambda: vkv.prompt_attn(**{**PROMPT, "ws_bytes": need - 1}), vkv.BUFFER_TOO_SMALL, "workspace")
    assert vkv.prompt_attn_workspace(vkv.BF16, 2, 100, 8, 128) < need
    assert vkv.prompt_attn_workspace(vkv.Q8_0, 2, 100, 8, 128) == 0
    assert vkv.prompt_attn_workspace(vkv.F32, 2, 100, 8, 96) == 0


LOGPROBS = dict(dtype=vkv.F32, logits=A, n_rows=2, n_vocab=1000, tokens=A, logprob=A, entropy=A, n_top=5, top_ids=A,
                top_logprobs=A, ws=A, ws_bytes=1 << 30)


@pytest.mark.parametrize("change", [
    dict(dtype=vkv.Q8_0), dict(logits=0), dict(logits=A + 4), dict(n_rows=-1), dict(n_rows=65536), dict(n_vocab=0),
    dict(n_vocab=1 << 31), dict(tokens=0), dict(logprob=0), dict(n_top=-1), dict(n_top=33), dict(n_top=20, n_vocab=19),
    dict(top_ids=0), dict(top_logprobs=0), dict(row_stride=999), dict(ws=0), dict(ws=A + 8), dict(entropy=A + 2)])
def test_logprobs_refuses(change):
    refused(lambda: vkv.logprobs(**{**LOGPROBS, **change}), text="log probabilities")


def test_logprobs_workspace():
    need = vkv.logprobs_workspace(2, 1000, 5)
    assert need > 0
    refused(lambda: vkv.logprobs(**{**LOGPROBS, "ws_bytes": 15}), vkv.BUFFER_TOO_SMALL, "workspace")
    assert vkv.logprobs_workspace(2, 1000, 33) == 0
    assert vkv.logprobs_workspace(-1, 1000, 3) == 0


def large_enough(call):
    """the size is accepted: the missing pointer, looked at next, is what the call refuses"""
    refused(call, vkv.INVALID_ARGUMENT, "workspace null")


def test_a_workspace_does_for_smaller_batches():
    for heads, kv in ((32, 8), (32, 32), (16, 1), (9, 3)):
        p = pages(n_pages=100000, n_kv_heads=kv)
        for most, longest in ((19, 8192), (64, 8192), (200, 1000), (1100, 300), (3, 100000)):
            need = vkv.paged_attn_workspace(p, most, heads, longest)
            for rows in {1, 2, 3, 5, 8, 16, 17, 18, 63, most // 2, most - 1, most}:
                for max_len in {257, 300, 1000, longest // 3, longest - 1, longest}:
                    for window in (0, 1, 255, 256, 1000, longest - 1):
                        # (a plan of one chunk needs none and refuses nothing here)
                        span = min(max_len, window + 31) if window else max_len
                        if not 0 < rows <= most or max_len > longest or span <= 1024:
                            continue
                        large_enough(lambda: vkv.paged_attn(p, 0, A, 8192, A, rows, max_len, vkv.F32, A, A, heads, 0.1,
                                                            window, 0, need))
    for most, vocab, top in ((17, 131072, 5), (251, 131072, 20), (64, 32003, 32), (2000, 5001, 32), (65535, 300, 3), (3, 1 << 30, 1)):
        need = vkv.logprobs_workspace(most, vocab, top)
        for rows in {1, 2, 3, 7, 8, 16, 31, 64, 200, most // 2, most - 1, most}:
            for fewer in {0, 1, top // 2, top}:
                for dtype in (vkv.F32, vkv.BF16):
                    for stride in (0, vocab + 1, vocab + 8):
                        if 0 < rows <= most:
                            large_enough(lambda: vkv.logprobs(dtype, A, rows, vocab, A, A, A, fewer, A, A, 0, need, row_stride=stride))
    for dtype in (vkv.F32, vkv.F16):
        need = vkv.prompt_attn_workspace(dtype, 9, 5000, 8, 128)
        for seqs in (1, 4, 9):
            for tokens in (1, 63, 1000, 5000):
                large_enough(lambda: vkv.prompt_attn(dtype, A, A, A, A, seqs, tokens, 32, 8, 128, 0.1, 0, A, 0, need))


def test_empty_calls_do_nothing():
    vkv.pages_append(pages(), 0, 0, 0, vkv.F32, 0, 0)
    vkv.paged_attn(pages(), **{**ATTN, "n_rows": 0})
    vkv.prompt_attn(**{**PROMPT, "n_seq": 0, "ws": 0, "ws_bytes": 0})
    vkv.prompt_attn(**{**PROMPT, "n_tokens": 0, "ws": 0, "ws_bytes": 0})
    vkv.logprobs(**{**LOGPROBS, "n_rows": 0})


def test_pages_struct_matches_the_header(tmp_path):
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    fields = [f for f, _ in vkv.Pages._fields_]
    src = tmp_path / "p.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "vkv.h"\nint main(void){printf("%zu\\n", sizeof(vkv_pages));'
                   + "".join(f'printf("%zu\\n", offsetof(vkv_pages, {f}));' for f in fields)
                   + f'printf("%d %d %d %d\\n", VKV_DTYPE_E4M3, VKV_DTYPE_I8, VKV_DTYPE_BF16, VKV_LOGPROBS_MAX_TOP);return 0;}}')
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(root, "include"), str(src), "-o", str(tmp_path / "p")], check=True)
    got = subprocess.run([str(tmp_path / "p")], capture_output=True, text=True, check=True).stdout.split()
    assert [int(x) for x in got] == ([ctypes.sizeof(vkv.Pages)] + [getattr(vkv.Pages, f).offset for f in fields]
                                     + [vkv.E4M3, vkv.I8, vkv.BF16, 32])
