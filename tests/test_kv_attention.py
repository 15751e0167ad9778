"""Attention over the paged KV pool and eviction from it: argument checks on the CPU, and on the GPU
every operator against its definition in 64 bits at the lengths, masks and layouts where it can go wrong."""
import math

import numpy as np
import pytest
import torch

import kvtools
from tensorcast_b200 import _native
from tensorcast_b200.kvattention import KvAttention, KvEvict
from tensorcast_b200.kvcache import KvGatherHash, KvWorkload

BF16, FP16 = torch.bfloat16, torch.float16


# ---------------------------------------------------------------- argument checks (CPU)

def refused(match, call):
    with pytest.raises(_native.TcxInvalidArgument, match=match):
        call()


def test_attention_refuses_what_it_cannot_run():
    w, _ = kvtools.tables([5, 40])
    make = lambda w=w, q=4, k=2, d=BF16, **kw: (lambda: KvAttention(w, q, k, d, **kw))  # noqa: E731
    refused("dtype", make(d=torch.float32))
    refused("multiple of kv_heads", make(q=5))
    refused("multiple of kv_heads", make(q=0))
    refused("64 or 128", make(k=1, q=2, w=kvtools.tables([5], kv_heads=3, dim=32)[0]))
    refused("multiple of 8", make(w=kvtools.tables([5], page=12)[0]))
    refused("layers x", make(w=kvtools.tables([5], planes=3)[0]))
    refused("negative", make(window=-1))
    refused("negative", make(sinks=-1))
    for scale in (0.0, -1.0, math.inf, math.nan):
        refused("scale", make(scale=scale))
    refused("query_tokens", make(query_tokens=[1]))
    refused("query_tokens", make(query_tokens=[1, -1]))
    refused("without prefix_pages", make(prefix_tokens=3))
    refused("prefix pages hold 16", make(prefix_pages=[1], prefix_tokens=17))
    refused("CUDA device", make(device="cpu"))
    bad = kvtools.tables([5, 40])[0]
    bad.seq_tokens[1] = 49
    refused("more tokens than its pages", make(w=bad))
    bad = kvtools.tables([5, 40])[0]
    bad.page_offsets[1] = 9
    refused("not decrease", make(w=bad))
    bad = kvtools.tables([5, 40])[0]
    bad.page_table = bad.page_table[:-1]
    refused("page table has", make(w=bad))


def test_evict_refuses_what_it_cannot_run():
    w, free = kvtools.tables([5, 40], taken=4)
    page = lambda *slots, n=(5, 20): KvWorkload(w.planes, w.pool_pages, 16, w.token_bytes,  # noqa: E731
                                                np.array(n, np.uint32), np.array([0, 1, 3], np.uint64),
                                                np.array(slots, np.uint32))
    good = page(*free[:3])
    make = lambda dst, k=2, **kw: (lambda: KvEvict(w, dst, k, **kw))  # noqa: E731
    refused("listed twice", make(page(free[0], free[1], free[0])))
    refused("is a source page", make(page(free[0], free[1], w.page_table[2])))
    refused("below sinks", make(good, sinks=3, recent=18))   # 21 of 40 tokens; 5 of 5 would stay
    refused("negative", make(good, sinks=-1))
    refused("same pool", make(kvtools.tables([5], taken=4)[0]))
    refused("multiple of 16", make(good, k=7))
    refused("more tokens than its pages", make(page(*free[:3], n=(17, 20))))
    refused("CUDA device", make(good, device="cpu"))


def test_page_slots_that_32_bits_do_not_hold_are_refused():
    """A slot of 2^32 + 3 is not slot 3. (-1 is a usual mark of an unused entry and stays outside of every pool.)"""
    w, free = kvtools.tables([5, 40], taken=3)
    wide = lambda slot: KvWorkload(**{**w.__dict__, "page_table": np.concatenate(  # noqa: E731
        [[slot], w.page_table[1:].astype(np.int64)])})
    for slot in (1 << 32, (1 << 32) + 3, -(1 << 32) + 3, -(1 << 31) - 1):
        refused("slot .* 32 bits", lambda: KvAttention(wide(slot), 4, 2, device="cpu"))
        refused("slot .* 32 bits", lambda: KvAttention(w, 4, 2, prefix_pages=[1, slot], prefix_tokens=3, device="cpu"))
        refused("slot .* 32 bits", lambda: KvEvict(wide(slot), w, 2, device="cpu"))
        refused("slot .* 32 bits", lambda: KvEvict(w, wide(slot), 2, device="cpu"))
    refused("CUDA device", lambda: KvAttention(wide(-1), 4, 2, device="cpu"))


def test_pieces_of_a_range_follow_from_the_lengths(tmp_path):
    """Warps that meet at a piece's end count the pieces by this where they cannot read the notes: it must say what
    the notes do, at every tile of every range."""
    import ctypes
    import os
    import subprocess
    csrc = os.path.join(os.path.dirname(_native.__file__), "csrc")
    (tmp_path / "pieces.cc").write_text("""
#include "kv_pieces.h"
extern "C" int ends(const uint32_t* tiles, uint32_t seq, uint32_t tile, uint32_t count, uint32_t i) {
  const tcx::TileEnd e = tcx::tile_end(seq, tile, count, i, [&](uint32_t s) { return tiles[s]; });
  return e.last + 2 * e.whole;
}""")
    so = str(tmp_path / "pieces.so")
    subprocess.check_call(["g++", "-std=c++17", "-shared", "-fPIC", "-I", csrc, str(tmp_path / "pieces.cc"), "-o", so])
    ends = ctypes.CDLL(so).ends
    rng = np.random.default_rng(0)
    for ranges in (1, 2, 3, 7, 20):
        tiles = rng.choice([0, 0, 1, 1, 2, 3, 9], 25).astype(np.uint32)
        tiles[-1] = 1
        flat = [(s, t) for s, n in enumerate(tiles) for t in range(n)]
        for r in range(ranges):
            mine = flat[len(flat) * r // ranges: len(flat) * (r + 1) // ranges]
            for i, (s, t) in enumerate(mine):
                last = i + 1 == len(mine) or mine[i + 1][0] != s
                whole = last and sum(x[0] == s for x in mine) == tiles[s]
                got = ends(tiles.ctypes.data_as(ctypes.c_void_p), int(mine[0][0]), mine[0][1], len(mine), i)
                assert got == last + 2 * whole, (ranges, r, i)


def test_negative_lengths_are_refused():
    """They would count as more than 2^31 tokens, which the device cuts to the pages' capacity."""
    w, free = kvtools.tables([5, 40], taken=3)
    bad = KvWorkload(**{**w.__dict__, "seq_tokens": np.array([5, -1])})
    refused("negative", lambda: KvAttention(bad, 4, 2, device="cpu"))
    refused("negative", lambda: KvEvict(bad, w, 2, device="cpu"))
    refused("negative", lambda: KvEvict(w, bad, 2, device="cpu"))


def test_windows_and_sinks_beyond_every_length_are_refused_at_once():
    """2^64 + 3 must not become 3 on its way to the entry point."""
    w, _ = kvtools.tables([5, 40])
    for size in (1 << 30, (1 << 64) + 3):
        refused("below 2\\^30", lambda: KvAttention(w, 4, 2, window=size, device="cpu"))
        refused("below 2\\^30", lambda: KvAttention(w, 4, 2, sinks=size, device="cpu"))


def attention_args(**kw):
    """Arguments that pass the checks of the C entry, made-up pointers among them, with `kw` changed."""
    a = _native.KvAttentionArgs(
        d_pool=0x1000, planes=2, pool_pages=8, page_tokens=16, kv_heads=2, q_heads=4, head_dim=64, dtype=0, k_plane=0,
        v_plane=1, d_page_table=0x1000, d_page_offsets=0x1000, d_seq_tokens=0x1000, n_seq=1, d_q_offsets=0x1000,
        q_tokens=1, max_q=1, total_pages=4, max_pages=4, scale=1.0, d_q=0x1000, q_token_stride=256, q_head_stride=64,
        d_out=0x2000, out_token_stride=256, out_head_stride=64, d_lse=0x1000, d_status=0x1000, d_counters=0x1000)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,message", [
    (dict(d_pool=None), "null device pointer"), (dict(d_lse=None), "null device pointer"),
    (dict(d_counters=None), "null device pointer"),
    (dict(d_page_table=None), "null device pointer"), (dict(planes=0), "must be > 0"),
    (dict(page_tokens=12), "multiple of 8"), (dict(head_dim=96), "head_dim"), (dict(dtype=2), "dtype"),
    (dict(q_heads=5), "multiple of kv_heads"), (dict(v_plane=2), "planes of the pool"),
    (dict(pool_pages=1 << 31), "2\\^31"), (dict(pool_pages=1 << 27), "2\\^31"), (dict(n_seq=70000), "65535"),
    (dict(q_tokens=1 << 30), "2\\^31"), (dict(max_q=2), "inconsistent"), (dict(max_pages=5), "inconsistent"),
    (dict(window=1 << 30), "2\\^30"), (dict(scale=0.0), "scale"), (dict(scale=math.nan), "scale"),
    (dict(scale=math.inf), "scale"), (dict(d_q=0x1008), "aligned"), (dict(q_head_stride=65), "strides"),
    (dict(d_prefix_table=0x1000), "null device pointer"),
    (dict(d_prefix_table=0x1000, d_prefix_tokens=0x1000, d_weights=0x1000), "shared prefix"),
])
def test_attention_entry_checks(change, message):
    import ctypes
    with pytest.raises(_native.TcxInvalidArgument, match=message):
        _native.call("tcx_kv_attention", ctypes.byref(attention_args(**change)), None, 0, None)


def test_attention_entry_checks_its_scratch():
    import ctypes
    L = _native.lib()
    for change in ({}, dict(d_prefix_table=0x1000, d_prefix_tokens=0x1000, prefix_pages=1), dict(max_q=9, q_tokens=9),
                   dict(d_weights=0x1000)):
        a = attention_args(**change)
        need = L.tcx_kv_attention_scratch_bytes(ctypes.byref(a))
        assert need > 0
        for scratch, size in ((None, need), (0x1000, need - 1), (0x1010, need)):
            with pytest.raises(_native.TcxInvalidArgument, match=f"scratch of {need} bytes"):
                _native.call("tcx_kv_attention", ctypes.byref(a), scratch, size, None)
    assert L.tcx_kv_attention_scratch_bytes(ctypes.byref(attention_args(head_dim=96))) == 0
    assert L.tcx_kv_attention_scratch_bytes(None) == 0


def test_attention_entry_without_work():
    import ctypes
    _native.call("tcx_kv_attention", ctypes.byref(attention_args(n_seq=0)), None, 0, None)
    _native.call("tcx_kv_attention", ctypes.byref(attention_args(q_tokens=0)), None, 0, None)
    with pytest.raises(_native.TcxInvalidArgument, match="null arguments"):
        _native.call("tcx_kv_attention", None, None, 0, None)


@pytest.mark.parametrize("change,message", [
    (dict(d_pool=None), "null device pointer"), (dict(d_keep=None), "null device pointer"),
    (dict(planes=3), "even"), (dict(page_tokens=0), "> 0"), (dict(head_bytes=24), "multiple of 16"),
    (dict(n_seq=70000), "65535"), (dict(dst_total_pages=1 << 28), "2\\^31"), (dict(d_pool=0x1008), "aligned"),
])
def test_evict_entry_checks(change, message):
    import ctypes
    a = _native.KvEvictArgs(
        d_pool=0x1000, planes=2, pool_pages=8, page_tokens=16, kv_heads=2, head_bytes=128, d_page_table=0x1000,
        d_page_offsets=0x1000, d_seq_tokens=0x1000, d_dst_page_table=0x1000, d_dst_page_offsets=0x1000,
        d_budgets=0x1000, n_seq=1, dst_total_pages=2, d_weights=0x1000, d_keep=0x1000, d_dst_weights=0x1000,
        d_dst_tokens=0x1000, d_status=0x1000)
    for k, v in change.items():
        setattr(a, k, v)
    with pytest.raises(_native.TcxInvalidArgument, match=message):
        _native.call("tcx_kv_evict", ctypes.byref(a), None)


# ---------------------------------------------------------------- attention (GPU)

def check(got, ref, dtype, longest):
    (out, lse), (want, want_lse, *_) = got, ref
    tol, tol_lse, _ = kvtools.bounds(ref, dtype, longest)
    empty = want_lse == -math.inf
    assert (lse[empty] == -math.inf).all() and (out[empty] == 0).all()
    assert ((lse.double() - want_lse).abs() <= tol_lse)[~empty].all(), (lse.double() - want_lse)[~empty].abs().max()
    off = (out.double() - want).abs()
    assert (off <= tol).all(), float((off / tol).max())


def queries(total, heads, dim, dtype, seed, scale=1.5):
    g = torch.Generator().manual_seed(seed + 100)
    return (torch.randn((total, heads, dim), generator=g) * scale).to(dtype).cuda()


def run(tokens, counts, *, kv_heads=2, group=4, dim=128, dtype=BF16, page=16, window=0, sinks=0, planes=2, layer=0,
        scale=None, seed=0, fill=math.nan, prefix=None, spare=0):
    """One call against the definition; everything outside the sequences' tokens holds `fill`."""
    taken = 0 if prefix is None else -(-prefix // page)
    w, free = kvtools.tables(tokens, page, kv_heads, dim, planes, spare, seed, taken=taken)
    pool = kvtools.make_pool(w, kv_heads, dim, dtype, seed, fill)
    more, rows = {}, None
    if prefix is not None:
        slots = free[:taken]
        at = np.arange(prefix)
        rows = slots[at // page].astype(np.int64) * page + at % page
        g = torch.Generator().manual_seed(seed + 7)
        pool[:, torch.from_numpy(rows)] = torch.randn((planes, prefix, kv_heads, dim), generator=g).to(dtype)
        more = {"prefix_pages": slots, "prefix_tokens": prefix}
    pool = pool.cuda()
    q = queries(sum(counts), kv_heads * group, dim, dtype, seed)
    att = KvAttention(w, kv_heads * group, kv_heads, dtype, query_tokens=counts, window=window, sinks=sinks,
                      scale=scale, **more)
    got = att.run(pool, layer, q)
    att.check_status()
    ref = kvtools.attention(w, pool, layer, q, counts, window, sinks, scale, rows)
    check(got, ref, dtype, max(tokens) + (prefix or 0))
    return att, pool, q, got, ref


LENGTHS = [1, 0, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300, 1000]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("kv_heads,group,dim,page", [(2, 4, 128, 16), (1, 1, 64, 8), (3, 5, 64, 24), (8, 8, 128, 64),
                                                     (1, 16, 128, 128), (2, 7, 128, 40), (1, 33, 64, 16)])
def test_decode(cuda_device, dtype, kv_heads, group, dim, page):
    run(LENGTHS, [1] * len(LENGTHS), kv_heads=kv_heads, group=group, dim=dim, page=page, dtype=dtype, planes=4,
        layer=1)


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 4), (16, 0), (64, 3), (100, 65), (128, 130), (5000, 2), (0, 9)])
@pytest.mark.parametrize("dim", [64, 128])
def test_decode_window_and_sinks(cuda_device, window, sinks, dim):
    run(LENGTHS, [1] * len(LENGTHS), dim=dim, window=window, sinks=sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("group,count", [(16, 1), (17, 1), (5, 4), (8, 4), (31, 1), (32, 1), (11, 3)])
def test_decode_around_the_rows_of_a_tile(cuda_device, dim, group, count):
    """Up to and beyond 16 and 32 rows, several short sequences to a range of work, parts to join, weights."""
    tokens = [1, 70, 0, 300, 5, 64, 129, 2000, 33, 12]
    att, pool, q, _, ref = run(tokens, [count] * len(tokens), kv_heads=2, group=group, dim=dim)
    run(tokens, [count] * len(tokens), kv_heads=1, group=group, dim=dim, window=90, sinks=7, dtype=FP16)
    weights = torch.zeros((2, att.weight_columns), device="cuda")
    att.run(pool, 0, q, weights=weights)
    relative = float(kvtools.bounds(ref, BF16, 2000)[2].max()) + 32 * 2.0 ** -24
    for s, n in enumerate(tokens):
        c = int(att.w.page_offsets[s]) * 16
        assert ((weights[:, c:c + n].double() - ref[2][s]).abs() <= relative * ref[2][s] + 2.0 ** -126).all(), s


@pytest.mark.gpu
def test_decode_one_long_sequence(cuda_device):
    run([20011], [1], kv_heads=1)
    run([20011, 3], [1, 1], kv_heads=1, window=9000, sinks=5, dtype=FP16)


@pytest.mark.gpu
@pytest.mark.parametrize("counts", [[2] * 14, [0, 1, 2, 3, 4, 0, 6, 7, 8, 9, 1, 1, 2, 0]])
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 3)])
@pytest.mark.parametrize("group", [1, 4, 6])
def test_several_queries(cuda_device, counts, window, sinks, group):
    """Speculated tokens; sequences without a query, and queries that stand before the first token and see nothing."""
    run(LENGTHS, counts, group=group, window=window, sinks=sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kv_heads,group,dim,page,window,sinks", [
    (BF16, 2, 4, 128, 16, 0, 0), (BF16, 1, 8, 64, 8, 100, 4), (FP16, 2, 1, 128, 24, 0, 0), (FP16, 1, 3, 64, 64, 1, 0),
    (BF16, 1, 5, 128, 256, 300, 129), (BF16, 1, 2, 128, 32, 129, 1)])
def test_prompts(cuda_device, dtype, kv_heads, group, dim, page, window, sinks):
    tokens = [1, 0, 2, 127, 128, 130, 513]
    run(tokens, tokens, kv_heads=kv_heads, group=group, dim=dim, page=page, dtype=dtype, window=window, sinks=sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", [(0, 0), (200, 4)])
def test_prompt_chunk_of_a_long_cache(cuda_device, window, sinks):
    run([3001, 40], [90, 40], kv_heads=1, window=window, sinks=sinks)
    run([700, 10, 65], [70, 33, 64], kv_heads=1, group=16, window=window, sinks=sinks)


@pytest.mark.gpu
def test_more_queries_than_tokens(cuda_device):
    """Queries that stand before the first token see nothing."""
    run([3, 0, 5], [70, 65, 5], kv_heads=1, group=3)


@pytest.mark.gpu
@pytest.mark.parametrize("prefix", [0, 1, 63, 128, 1000])
@pytest.mark.parametrize("counts", [[1] * 9, [1, 0, 2, 5, 1, 1, 3, 1, 40]])
def test_shared_prefix(cuda_device, prefix, counts):
    run([0, 1, 2, 16, 17, 64, 129, 5, 300], counts, prefix=prefix, dtype=FP16)


@pytest.mark.gpu
@pytest.mark.parametrize("group,dim,batch", [(1, 64, 3), (8, 128, 40), (5, 128, 70)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (150, 4), (20, 300)])
def test_shared_prefix_batches(cuda_device, group, dim, batch, window, sinks):
    tokens = [(7 * i) % 200 for i in range(batch)]
    run(tokens, [1] * batch, kv_heads=2, group=group, dim=dim, prefix=515, window=window, sinks=sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 4), (350, 310), (1, 0)])
@pytest.mark.parametrize("group,dim", [(4, 64), (1, 128)])
def test_shared_prefix_with_prompts(cuda_device, window, sinks, group, dim):
    """Many queries behind a prefix, some standing inside it, the windows reaching back across its end."""
    run([0, 50, 130, 7, 260], [3, 50, 70, 12, 260], kv_heads=2, group=group, dim=dim, prefix=301, window=window,
        sinks=sinks)


@pytest.mark.gpu
def test_lengths_of_the_prefix_and_the_sequences_may_change(cuda_device):
    w, free = kvtools.tables([40, 5], spare=2, taken=12)
    pool = kvtools.make_pool(w, 2, 64, BF16).cuda()
    q = queries(2, 8, 64, BF16, 0)
    att = KvAttention(w, 8, 2, prefix_pages=free[:12], prefix_tokens=100)
    for prefix, tokens in ((100, [40, 5]), (0, [0, 21]), (1, [1, 0]), (192, [70, 33])):
        att.prefix_tokens.fill_(prefix)
        att.seq_tokens.copy_(torch.tensor(tokens, dtype=torch.int32))
        rows = free[:12][np.arange(prefix) // 16].astype(np.int64) * 16 + np.arange(prefix) % 16
        check(att.run(pool, 0, q), kvtools.attention(w, pool, 0, q, [1, 1], prefix_rows=rows, tokens=tokens), BF16, 300)
    att.check_status()
    att.prefix_tokens.fill_(193)
    att.run(pool, 0, q)
    with pytest.raises(_native.TcxError, match="more tokens"):
        att.check_status()


@pytest.mark.gpu
def test_large_scores_and_small_scale(cuda_device):
    run(LENGTHS, [1] * len(LENGTHS), scale=3.0)
    run([300], [300], kv_heads=1, scale=3.0)
    run(LENGTHS, [1] * len(LENGTHS), scale=1e-30)


@pytest.mark.gpu
@pytest.mark.parametrize("fill", [math.inf, -math.inf, math.nan])
def test_values_that_no_query_sees_do_not_matter(cuda_device, fill):
    """Behind the sequences' ends, in spare pages, and between the sinks and the window."""
    tokens, window, sinks = [5, 64, 130, 400, 1000], 70, 5
    w, _ = kvtools.tables(tokens, spare=2)
    pool = kvtools.make_pool(w, 2, 64, BF16, fill=fill)
    for s, n in enumerate(tokens):
        hidden = kvtools.token_rows(w, s)[sinks:max(n - window, sinks)]
        pool[:, torch.from_numpy(hidden)] = fill
    pool, q = pool.cuda(), queries(len(tokens), 8, 64, BF16, 0)
    got = KvAttention(w, 8, 2, window=window, sinks=sinks).run(pool, 0, q)
    check(got, kvtools.attention(w, pool, 0, q, [1] * 5, window, sinks), BF16, 1000)


@pytest.mark.gpu
def test_non_finite_values_that_a_query_sees_show(cuda_device):
    w, _ = kvtools.tables([40, 40, 40])
    pool = kvtools.make_pool(w, 2, 64, BF16)
    pool[1, kvtools.token_rows(w, 0)[7]] = math.inf
    pool[0, kvtools.token_rows(w, 1)[9]] = math.nan
    q = queries(3, 4, 64, BF16, 0)
    out, lse = KvAttention(w, 4, 2).run(pool.cuda(), 0, q)
    assert (out[0] == math.inf).all() and torch.isfinite(lse[0]).all()
    assert torch.isnan(out[1]).all() and torch.isnan(lse[1]).all()
    assert torch.isfinite(out[2]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("counts", [[1, 1, 1], [40, 3, 100]])
def test_strided_queries_and_padding_rows(cuda_device, counts):
    tokens = [100, 17, 400]
    w, _ = kvtools.tables(tokens, kv_heads=2, dim=64)
    pool = kvtools.make_pool(w, 2, 64, BF16).cuda()
    n = sum(counts)
    fused = torch.randn((n + 5, 12 * 64), device="cuda").to(BF16)
    q = fused[:, : 8 * 64].unflatten(1, (8, 64))
    att = KvAttention(w, 8, 2, query_tokens=counts)
    ref = kvtools.attention(w, pool, 0, q[:n], counts)
    out, lse = att.run(pool, 0, q)
    check((out[:n], lse[:n]), ref, BF16, 400)
    assert (out[n:] == 0).all() and (lse[n:] == 0).all()
    # heads outside, tokens inside: the given buffers' rows behind the last sequence stay as they were
    qt = q.transpose(0, 1).contiguous().transpose(0, 1)
    ot = torch.full((8, n + 5, 64), 7.0, dtype=BF16, device="cuda").transpose(0, 1)
    lt = torch.full((n + 5, 8), 7.0, device="cuda")
    got, got_lse = att.run(pool, 0, qt, out=ot, lse=lt)
    assert got.data_ptr() == ot.data_ptr() and (ot[:n] == out[:n]).all() and (lt[:n] == lse[:n]).all()
    assert (ot[n:] == 7).all() and (lt[n:] == 7).all()


@pytest.mark.gpu
def test_pages_may_be_listed_more_than_once(cuda_device):
    """Two sequences that share their first pages."""
    w, _ = kvtools.tables([100, 90])
    w.page_table[int(w.page_offsets[1]):int(w.page_offsets[1]) + 3] = w.page_table[:3]
    pool = kvtools.make_pool(w, 2, 64, BF16).cuda()
    q = queries(2, 4, 64, BF16, 0)
    check(KvAttention(w, 4, 2).run(pool, 0, q), kvtools.attention(w, pool, 0, q, [1, 1]), BF16, 100)


@pytest.mark.gpu
@pytest.mark.parametrize("counts", [[1, 1], [70, 30]])
def test_bad_tables_are_reported(cuda_device, counts):
    w, _ = kvtools.tables([100, 90])
    pool = kvtools.make_pool(w, 2, 64, BF16).cuda()
    q = queries(sum(counts), 4, 64, BF16, 0)
    bad = KvWorkload(**{**w.__dict__, "page_table": w.page_table.copy()})
    bad.page_table[2] = 10_000_000
    att = KvAttention(bad, 4, 2, query_tokens=counts)
    out, _ = att.run(pool, 0, q)
    with pytest.raises(_native.TcxError, match="outside the pool"):
        att.check_status()
    ref = kvtools.attention(w, pool, 0, q, counts)
    assert (out[counts[0]:].double() - ref[0][counts[0]:]).abs().max() < 0.05  # the other sequence is served
    att = KvAttention(w, 4, 2, query_tokens=counts)
    att.seq_tokens[1] = 1000
    att.run(pool, 0, q)
    with pytest.raises(_native.TcxError, match="more tokens"):
        att.check_status()


@pytest.mark.gpu
def test_run_refuses_what_it_cannot_take(cuda_device):
    w, _ = kvtools.tables([20, 30])
    pool = kvtools.make_pool(w, 2, 64, BF16).cuda()
    q = queries(2, 4, 64, BF16, 0)
    att = KvAttention(w, 4, 2)
    refused("layer 1", lambda: att.run(pool, 1, q))
    refused("layer -1", lambda: att.run(pool, -1, q))
    refused("pool has", lambda: att.run(pool[:1], 0, q))
    refused("contiguous", lambda: att.run(pool.transpose(0, 1), 0, q))
    refused("contiguous tensor on cuda", lambda: att.run(pool.cpu(), 0, q))
    refused("q must be torch.bfloat16", lambda: att.run(pool, 0, q.half()))
    refused("q must be torch.bfloat16", lambda: att.run(pool, 0, q.cpu()))
    refused("q must be \\[", lambda: att.run(pool, 0, q[:1]))
    refused("q must be \\[", lambda: att.run(pool, 0, q[:, :3]))
    refused("strides", lambda: att.run(pool, 0, torch.zeros((2, 4, 65), dtype=BF16, device="cuda")[:, :, :64]))
    refused("alignment", lambda: att.run(pool, 0, torch.zeros(2 * 4 * 64 + 1, dtype=BF16, device="cuda")[1:]
                                         .view(2, 4, 64)))
    refused("share memory", lambda: att.run(pool, 0, q, out=q))
    refused("lse", lambda: att.run(pool, 0, q, lse=torch.zeros((2, 4), dtype=FP16, device="cuda")))
    refused("no gradient", lambda: att.run(pool, 0, q.clone().requires_grad_()))
    refused("weights must be", lambda: att.run(pool, 0, q, weights=torch.zeros((2, 7), device="cuda")))
    shared = KvAttention(w, 4, 2, prefix_pages=[0], prefix_tokens=3)
    refused("shared prefix", lambda: shared.run(pool, 0, q, weights=torch.zeros((2, att.weight_columns),
                                                                               device="cuda")))


@pytest.mark.gpu
@pytest.mark.parametrize("counts,prefix", [([1] * 5, None), ([30] * 5, None), ([1] * 5, 300)])
def test_captured_calls_follow_the_lengths(cuda_device, counts, prefix):
    """A graph of two calls on one handle, replayed with other lengths and other queries."""
    tokens, page, taken = [200, 30, 31, 64, 90], 16, 0 if prefix is None else -(-prefix // 16)
    w, free = kvtools.tables(tokens, spare=6, dim=128, taken=taken)
    pool = kvtools.make_pool(w, 2, 128, BF16).cuda()
    more, rows = {}, None
    if prefix is not None:
        more = {"prefix_pages": free[:taken], "prefix_tokens": prefix}
        rows = free[:taken][np.arange(prefix) // page].astype(np.int64) * page + np.arange(prefix) % page
    q = queries(sum(counts), 8, 128, BF16, 0)
    att = KvAttention(w, 8, 2, query_tokens=counts, **more)
    att.run(pool, 0, q)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        one = att.run(pool, 0, q)
        two = att.run(pool, 0, q)
    for step in range(3):
        more_tokens = [n + 17 * step for n in tokens]
        att.seq_tokens.copy_(torch.tensor(more_tokens, dtype=torch.int32))
        q.copy_(queries(sum(counts), 8, 128, BF16, step))
        g.replay()
        torch.cuda.synchronize()
        ref = kvtools.attention(w, pool, 0, q, counts, prefix_rows=rows, tokens=more_tokens)
        check(one, ref, BF16, 600)
        assert (one[0] == two[0]).all() and (one[1] == two[1]).all()
    att.check_status()


@pytest.mark.gpu
def test_streams(cuda_device):
    """Calls of one handle on two streams at once, by stream object and by handle, give the same as one alone."""
    tokens = [3000, 100, 2000, 5]
    w, _ = kvtools.tables(tokens, dim=128)
    pool = kvtools.make_pool(w, 2, 128, BF16).cuda()
    q = queries(4, 8, 128, BF16, 0)
    att = KvAttention(w, 8, 2)
    want = att.run(pool, 0, q)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(20):
        got += [att.run(pool, 0, q, stream=a), att.run(pool, 0, q, stream=b.cuda_stream), att.run(pool, 0, q, stream=0)]
    torch.cuda.synchronize()
    for out, lse in got:
        assert (out == want[0]).all() and (lse == want[1]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("counts", [[1, 1, 1], [40, 1, 70]])
def test_pool_beyond_32_bit_offsets(cuda_device, counts):
    """Pages at the end of planes of 5.2 GB each, the second of two layers."""
    kv_heads, dim, page, pages = 8, 128, 16, 80_000
    tokens = [100, 33, 71]
    need = [-(-n // page) for n in tokens]
    slots = np.arange(pages - 40, pages, dtype=np.uint32)[::-1].copy()
    offs = np.concatenate([[0], np.cumsum(need)]).astype(np.uint64)
    w = KvWorkload(4, pages, page, kv_heads * dim * 2, np.array(tokens, np.uint32), offs, slots[: sum(need)])
    pool = torch.zeros((4, pages * page, kv_heads, dim), dtype=BF16, device="cuda")
    pool[:, -40 * page:] = torch.randn((4, 40 * page, kv_heads, dim), device="cuda").to(BF16)
    q = queries(sum(counts), 16, dim, BF16, 0)
    att = KvAttention(w, 16, kv_heads, query_tokens=counts)
    weights = torch.zeros((2, kv_heads, att.weight_columns), device="cuda")
    ref = kvtools.attention(w, pool, 1, q, counts)
    check(att.run(pool, 1, q, weights=weights[1]), ref, BF16, 100)
    for s, n in enumerate(tokens):
        c = int(offs[s]) * page
        assert (weights[1, :, c:c + n].double() - ref[2][s]).abs().max() < 1e-3
    dst = KvWorkload(4, pages, page, w.token_bytes, np.full(3, 20, np.uint32), np.array([0, 2, 4, 6], np.uint64),
                     slots[-6:].copy())
    keep, _, _ = KvEvict(w, dst, kv_heads).run(pool, weights)
    for s in range(3):
        idx = keep[1, 3, 32 * s: 32 * s + 20].cpu().numpy()
        want = pool[2:, torch.from_numpy(kvtools.token_rows(w, s)[idx]).cuda(), 3]
        assert (pool[2:, torch.from_numpy(kvtools.token_rows(dst, s)).cuda(), 3] == want).all()


@pytest.mark.gpu
def test_many_sequences(cuda_device):
    """More sequences than threads; most of them without queries or tokens."""
    rng = np.random.default_rng(0)
    tokens = rng.integers(0, 40, 3000).tolist()
    counts = rng.integers(0, 2, 3000).tolist()
    run(tokens, counts, kv_heads=1, group=2, dim=64)
    counts = [c * 9 for c in counts[:300]]
    run(tokens[:300], counts, kv_heads=1, group=2, dim=64)


@pytest.mark.gpu
def test_nothing_to_do(cuda_device):
    w, free = kvtools.tables([20, 30], taken=4)
    pool = kvtools.make_pool(w, 2, 64, BF16).cuda()
    out, lse = KvAttention(w, 4, 2, query_tokens=[0, 0]).run(pool, 0, queries(0, 4, 64, BF16, 0))
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    none = KvWorkload(2, w.pool_pages, 16, w.token_bytes, np.zeros(0, np.uint32), np.zeros(1, np.uint64),
                      np.zeros(0, np.uint32))
    out, lse = KvAttention(none, 4, 2).run(pool, 0, queries(0, 4, 64, BF16, 0))
    assert out.shape == (0, 4, 64)
    keep, left, tokens = KvEvict(none, none, 2).run(pool, torch.zeros((1, 2, 0), device="cuda"))
    assert keep.shape == left.shape == (1, 2, 0) and tokens.shape == (0,)
    # sequences with queries and without a page
    empty = KvWorkload(2, w.pool_pages, 16, w.token_bytes, np.zeros(2, np.uint32), np.zeros(3, np.uint64),
                       np.zeros(0, np.uint32))
    for counts in ([1, 2], [40, 2]):
        n = sum(counts)
        att = KvAttention(empty, 4, 2, query_tokens=counts)
        out, lse = att.run(pool, 0, queries(n, 4, 64, BF16, 0), weights=torch.zeros((2, 0), device="cuda"))
        att.check_status()
        assert (out == 0).all() and (lse == -math.inf).all()


@pytest.mark.gpu
def test_first_call_of_a_process_may_be_captured(cuda_device):
    import subprocess
    import sys
    code = """
import torch, kvtools
from tensorcast_b200.kvattention import KvAttention, KvEvict
from tensorcast_b200.kvcache import KvWorkload
import numpy as np
w, free = kvtools.tables([100, 30], taken=8)
pool = kvtools.make_pool(w, 2, 64, torch.bfloat16).cuda()
dst = KvWorkload(w.planes, w.pool_pages, 16, w.token_bytes, np.full(2, 20, np.uint32), np.array([0, 2, 4], np.uint64), free[:4])
for counts, more in (([1, 1], {}), ([60, 20], {}), ([1, 1], dict(prefix_pages=free[4:8], prefix_tokens=60))):
    q = torch.randn((sum(counts), 4, 64), device="cuda").bfloat16()
    att = KvAttention(w, 4, 2, query_tokens=counts, **more)
    weights = None if more else torch.zeros((2, att.weight_columns), device="cuda")
    ev = KvEvict(w, dst, 2)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, lse = att.run(pool, 0, q, weights=weights)
        if weights is not None:
            keep, _, _ = ev.run(pool, weights[None])
    g.replay()
    torch.cuda.synchronize()
    want, _ = att.run(pool, 0, q)
    assert (out == want).all()
    if weights is not None:
        again, _, _ = ev.run(pool, weights[None])
        assert (keep == again).all()
print("done")
"""
    import os
    here = os.path.dirname(os.path.abspath(__file__))
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([here, os.path.dirname(here)]))
    r = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "done" in r.stdout, r.stderr[-2000:]


# ---------------------------------------------------------------- the range of the probabilities (GPU)

def steered(scores, values, count, group, dim=64, seed=0):
    """A sequence of len(scores) fp16 tokens of one kv head whose scaled scores are about `scores` for every row
    (plus normal ones of size 0.1), its values, and its `count` queries."""
    n = len(scores)
    w, _ = kvtools.tables([n], kv_heads=1, dim=dim)
    pool = kvtools.make_pool(w, 1, dim, FP16)
    rows = torch.from_numpy(kvtools.token_rows(w, 0))
    g = torch.Generator().manual_seed(seed)
    k = torch.randn((n, dim), generator=g) * 0.1
    k[:, 0] = scores.float() * dim ** 0.5 / 4
    q = torch.randn((count, group, dim), generator=g)
    q[:, :, 0] = 4
    pool[0, rows, 0], pool[1, rows, 0] = k.half(), values.half()
    return w, pool.cuda(), q.half().cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("count", [1, 40])
@pytest.mark.parametrize("gap", [17.0, 19.0, 25.0])
@pytest.mark.parametrize("sink", [0.0, 2.0 ** -9, 1.0])
def test_fp16_tokens_far_below_a_strong_first_one_count(cuda_device, count, gap, sink):
    """A first token that takes nearly all of the softmax, and whose value may be small or 0: the 40000 others
    make up much of the output, though each weighs 2^-25 to 2^-36 of it."""
    g = torch.Generator().manual_seed(1)
    scores = torch.zeros(40000)
    scores[0] = gap
    values = torch.randn((40000, 64), generator=g).abs() * 8
    values[0] *= sink
    w, pool, q = steered(scores, values, count, 4)
    got = KvAttention(w, 4, 1, FP16, query_tokens=[count]).run(pool, 0, q)
    check(got, kvtools.attention(w, pool, 0, q, [count]), FP16, 40000)


@pytest.mark.gpu
@pytest.mark.parametrize("count", [1, 40])
@pytest.mark.parametrize("order", ["up", "down", "zigzag", "steps", "mixed"])
def test_fp16_scores_that_rise_and_fall_along_the_row(cuda_device, count, order):
    """Scores over a range of 2^26 in weight, with values that make every token count alike. A probability below
    2^-14 is off by 2^-25 where the largest of its 128 tokens has 2^-1 at least: by 2^-24 of that one's weight."""
    n = 3000
    at = torch.arange(n, dtype=torch.float64)
    z = {"up": at / n * 18, "down": 18 - at / n * 18, "zigzag": (at % 500 - 250).abs() / 250 * 18,
         "steps": (at // 128 % 2) * 18, "mixed": torch.rand(n, generator=torch.Generator().manual_seed(2)) * 18}[order]
    values = (torch.rand((n, 64), generator=torch.Generator().manual_seed(3)) + 0.5) * torch.exp(9 - z)[:, None]
    w, pool, q = steered(z - 9, values, count, 4)
    out, lse = KvAttention(w, 4, 1, FP16, query_tokens=[count]).run(pool, 0, q)
    ref = kvtools.attention(w, pool, 0, q, [count])
    tol, tol_lse, _ = kvtools.bounds(ref, FP16, n)
    rows = torch.from_numpy(kvtools.token_rows(w, 0)).cuda()
    k, v = pool[0, rows, 0].double(), pool[1, rows, 0].double()
    p = torch.exp((q.double() @ k.t()) / 8 - ref[1][..., None])
    see = torch.arange(n, device="cuda") <= n - count + torch.arange(count, device="cuda")[:, None]
    p = torch.nn.functional.pad(p * see[:, None], (0, -n % 128)).unflatten(-1, (-1, 128))
    size = torch.nn.functional.pad(v.abs(), (0, 0, 0, -n % 128)).unflatten(0, (-1, 128)).sum(1)
    tol = tol + 2.0 ** -24 * p.amax(-1) @ size
    assert ((out.double() - ref[0]).abs() <= tol).all(), float(((out.double() - ref[0]).abs() / tol).max())
    assert ((lse.double() - ref[1]).abs() <= tol_lse).all()


@pytest.mark.gpu
@pytest.mark.parametrize("gap", [17.0, 19.0, 25.0])
def test_fp16_tail_of_a_decode_batch(cuda_device, gap):
    """The same for one query token, in sequences that share their pages: a warp goes through many tiles of each."""
    n, batch = 20000, 60
    values = torch.randn((n, 64), generator=torch.Generator().manual_seed(1)).abs() * 8
    values[0] = 0
    scores = torch.zeros(n)
    scores[0] = gap
    one, pool, q = steered(scores, values, 1, 4)
    pages = len(one.page_table)
    w = KvWorkload(2, one.pool_pages, 16, one.token_bytes, np.full(batch, n, np.uint32),
                   (np.arange(batch + 1) * pages).astype(np.uint64), np.tile(one.page_table, batch))
    out, lse = KvAttention(w, 4, 1, FP16).run(pool, 0, q.expand(batch, 4, 64))
    ref = kvtools.attention(one, pool, 0, q, [1])
    for s in range(batch):
        check((out[s:s + 1], lse[s:s + 1]), ref, FP16, n)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("group,dim,batch", [(4, 64, 4), (8, 128, 40), (5, 128, 70), (8, 64, 64)])
def test_prefix_values_that_one_sequence_sees_stay_out_of_the_others(cuda_device, dtype, group, dim, batch):
    """Windows that reach back into a shared prefix from different places, and queries that stand inside it: an
    infinite or NaN value in the prefix shows in the rows that see it, in its column, and nowhere else."""
    prefix, window, sinks, page = 515, 150, 4, 16
    tokens = [(37 * i) % 190 + 10 * (i % 3) for i in range(batch)]
    counts = [1 if i % 5 else 1 + 7 * i % 33 for i in range(batch)] if batch > 4 else [1] * batch
    taken = -(-prefix // page)
    w, free = kvtools.tables(tokens, page, 2, dim, taken=taken)
    pool = kvtools.make_pool(w, 2, dim, dtype)
    rows = free[:taken][np.arange(prefix) // page].astype(np.int64) * page + np.arange(prefix) % page
    g = torch.Generator().manual_seed(7)
    pool[:, torch.from_numpy(rows)] = torch.randn((2, prefix, 2, dim), generator=g).to(dtype)
    for token, column, value in ((2, 1, math.inf), (380, 3, math.nan), (400, 4, -math.inf), (430, 5, math.inf),
                                 (440, 6, math.inf), (441, 6, -math.inf), (500, 7, math.inf), (511, 8, math.nan),
                                 (512, 9, -math.inf), (514, 10, math.inf), (300, 11, math.nan)):
        pool[1, int(rows[token]), token % 2, column] = value
    pool, q = pool.cuda(), queries(sum(counts), 2 * group, dim, dtype, 0)
    att = KvAttention(w, 2 * group, 2, dtype, query_tokens=counts, window=window, sinks=sinks,
                      prefix_pages=free[:taken], prefix_tokens=prefix)
    out, lse = att.run(pool, 0, q)
    att.check_status()
    ref = kvtools.attention(w, pool, 0, q, counts, window, sinks, prefix_rows=rows)
    finite = torch.isfinite(ref[0])
    assert finite.any() and not finite.all()
    assert (torch.isnan(out) == torch.isnan(ref[0])).all()
    assert (out[torch.isinf(ref[0])].double() == ref[0][torch.isinf(ref[0])]).all()
    tol, tol_lse, _ = kvtools.bounds(ref, dtype, 800)
    assert ((out.double() - ref[0]).abs() <= tol)[finite].all()
    assert ((lse.double() - ref[1]).abs() <= tol_lse)[ref[1] > -math.inf].all()


@pytest.mark.gpu
def test_check_status_waits_for_every_stream_and_starts_anew(cuda_device):
    """The error of a call that another stream still holds back is found; once it is raised, it is forgotten."""
    w, free = kvtools.tables([100, 90], taken=4)
    pool = kvtools.make_pool(w, 2, 64, BF16).cuda()
    q = queries(2, 4, 64, BF16, 0)
    dst = KvWorkload(w.planes, w.pool_pages, 16, w.token_bytes, np.array([20, 20], np.uint32),
                     np.array([0, 2, 4], np.uint64), free[:4].copy())
    weights = torch.ones((1, 2, int(w.page_offsets[-1]) * 16), device="cuda")
    side = torch.cuda.Stream()
    for handle, call in ((KvAttention(w, 4, 2), lambda h, s: h.run(pool, 0, q, stream=s)),
                         (KvEvict(w, dst, 2), lambda h, s: h.run(pool, weights, stream=s))):
        good = handle.page_table.clone()
        call(handle, side)
        handle.check_status()
        handle.page_table[1] = 10_000_000
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(300_000_000)
        call(handle, side)
        with pytest.raises(_native.TcxError, match="outside the pool"):
            handle.check_status()
        handle.page_table.copy_(good)
        handle.check_status()
        call(handle, None)
        handle.check_status()
        handle.seq_tokens[1] = 1000
        call(handle, None)
        with pytest.raises(_native.TcxError, match="more tokens"):
            handle.check_status()


@pytest.mark.gpu
def test_outputs_whose_rows_overlap_are_refused(cuda_device):
    w, _ = kvtools.tables([20, 30])
    pool = kvtools.make_pool(w, 2, 64, BF16).cuda()
    q = queries(2, 4, 64, BF16, 0)
    att = KvAttention(w, 4, 2)
    flat = torch.zeros(4096, dtype=BF16, device="cuda")
    for strides in ((0, 64, 1), (256, 0, 1), (256, 32, 1), (64, 64, 1), (192, 64, 1), (64, 120, 1)):
        refused("rows overlap", lambda: att.run(pool, 0, q, out=flat.as_strided((2, 4, 64), strides)))
    want = att.run(pool, 0, q)[0]
    for strides in ((256, 64, 1), (64, 128, 1), (320, 72, 1), (264, 64, 1)):
        assert (att.run(pool, 0, q, out=flat.as_strided((2, 4, 64), strides))[0] == want).all()


@pytest.mark.gpu
def test_strides_of_single_tokens_and_heads_do_not_matter(cuda_device):
    """The stride of an axis of one entry can be anything: a lone query row, one head, one kv head's weights."""
    w, _ = kvtools.tables([70], kv_heads=1)
    pool = kvtools.make_pool(w, 1, 64, BF16).cuda()
    q = queries(1, 1, 64, BF16, 0)
    att = KvAttention(w, 1, 1)
    columns = att.weight_columns
    want, got = torch.zeros((1, columns), device="cuda"), torch.zeros((columns, 1), device="cuda").t()
    assert got.stride() == (1, 1)
    out, lse = att.run(pool, 0, q, weights=want)
    odd = att.run(pool, 0, q.as_strided((1, 1, 64), (3, 5, 1)), weights=got,
                  out=torch.zeros(64, dtype=BF16, device="cuda").as_strided((1, 1, 64), (1, 1, 1)))
    assert (odd[0] == out).all() and (odd[1] == lse).all() and (got == want).all()


@pytest.mark.gpu
@pytest.mark.parametrize("count", [1, 40])
@pytest.mark.parametrize("where", ["prefix", "own"])
def test_non_finite_values_show_through_a_weight_of_zero(cuda_device, where, count):
    """A row sees a prefix and its own tokens, one of which weighs nothing in 32 bits beside the other."""
    prefix, n = 20, 60
    w, free = kvtools.tables([n], taken=2, kv_heads=1)
    pool = kvtools.make_pool(w, 1, 64, BF16)
    rows = free[:2][np.arange(prefix) // 16].astype(np.int64) * 16 + np.arange(prefix) % 16
    mine = kvtools.token_rows(w, 0)
    pool[0, torch.from_numpy(rows), :, 0] = 30.0 if where == "own" else -30.0
    pool[0, torch.from_numpy(mine), :, 0] = -30.0 if where == "own" else 30.0
    at = int(rows[7] if where == "prefix" else mine[7])
    pool[1, at, 0, 3], pool[1, at, 0, 4] = math.inf, math.nan
    q = queries(count, 4, 64, BF16, 0)
    q[:, :, 0] = 40.0
    out, lse = KvAttention(w, 4, 1, query_tokens=[count], prefix_pages=free[:2], prefix_tokens=prefix).run(pool.cuda(), 0, q)
    assert not torch.isfinite(out[..., 3:5]).any()
    assert torch.isfinite(out[..., :3]).all() and torch.isfinite(out[..., 5:]).all() and torch.isfinite(lse).all()


# ---------------------------------------------------------------- accumulated weights (GPU)

@pytest.mark.gpu
@pytest.mark.parametrize("counts", [[1] * 8, [2, 0, 1, 3, 9, 1, 70, 200]])
@pytest.mark.parametrize("window,sinks,group,dim,dtype", [(0, 0, 4, 128, BF16), (40, 3, 3, 64, FP16),
                                                          (0, 0, 16, 64, BF16)])
def test_weights(cuda_device, counts, window, sinks, group, dim, dtype):
    tokens = [1, 5, 0, 64, 200, 129, 300, 1000]
    w, _ = kvtools.tables(tokens, dim=dim, planes=4, spare=1)
    pool = kvtools.make_pool(w, 2, dim, dtype, fill=math.nan).cuda()
    q = queries(sum(counts), 2 * group, dim, dtype, 1)
    att = KvAttention(w, 2 * group, 2, dtype, query_tokens=counts, window=window, sinks=sinks)
    wide = torch.full((2, att.weight_columns + 3), 5.0, device="cuda")
    weights = wide[:, : att.weight_columns]
    start = torch.rand(weights.shape, device="cuda")
    weights.copy_(start)
    got = att.run(pool, 1, q, weights=weights)
    att.check_status()
    ref = kvtools.attention(w, pool, 1, q, counts, window, sinks)
    check(got, ref, dtype, 1000)
    relative = float(kvtools.bounds(ref, dtype, 1000)[2].max())
    for s, n in enumerate(tokens):
        c = int(w.page_offsets[s]) * 16
        want = start[:, c:c + n].double() + ref[2][s]
        rows = counts[s] * group
        assert ((weights[:, c:c + n].double() - want).abs()
                <= (relative + rows * 2.0 ** -24) * ref[2][s] + want * 2.0 ** -23).all(), s
        end = int(w.page_offsets[s + 1]) * 16
        assert (weights[:, c + n:end] == start[:, c + n:end]).all()
    assert (wide[:, att.weight_columns:] == 5).all()


@pytest.mark.gpu
@pytest.mark.parametrize("counts", [[1, 1], [300, 40]])
def test_weights_are_the_same_every_time(cuda_device, counts):
    w, _ = kvtools.tables([4000, 90], dim=128)
    pool = kvtools.make_pool(w, 2, 128, BF16).cuda()
    q = queries(sum(counts), 8, 128, BF16, 0)
    att = KvAttention(w, 8, 2, query_tokens=counts)
    seen = []
    for _ in range(3):
        weights = torch.zeros((2, att.weight_columns), device="cuda")
        out, lse = att.run(pool, 0, q, weights=weights)
        seen.append((out, lse, weights))
    for other in seen[1:]:
        assert all((a == b).all() for a, b in zip(seen[0], other))


# ---------------------------------------------------------------- eviction (GPU)

def evict_case(tokens, budgets, *, kv_heads=2, dim=64, layers=2, page=16, sinks=0, recent=0, seed=0, spare=0,
               weights=None):
    dst_pages = [-(-b // page) + spare for b in budgets]
    w, free = kvtools.tables(tokens, page, kv_heads, dim, 2 * layers, seed=seed, taken=sum(dst_pages))
    offs = np.concatenate([[0], np.cumsum(dst_pages)]).astype(np.uint64)
    dst = KvWorkload(w.planes, w.pool_pages, page, w.token_bytes, np.array(budgets, np.uint32), offs,
                     free[: sum(dst_pages)].copy())
    pool = kvtools.make_pool(w, kv_heads, dim, BF16, seed)
    if weights is None:
        weights = torch.rand((layers, kv_heads, int(w.page_offsets[-1]) * page),
                             generator=torch.Generator().manual_seed(seed))
    before = pool.clone()
    pool, dev = pool.cuda(), weights.cuda()
    ev = KvEvict(w, dst, kv_heads, sinks=sinks, recent=recent)
    keep, left, n = ev.run(pool, dev)
    ev.check_status()
    assert (dev.cpu().nan_to_num(-9) == weights.nan_to_num(-9)).all()
    want = before.clone()
    want_keep = np.full((layers, kv_heads, int(offs[-1]) * page), -1, np.int32)
    want_left = np.zeros(want_keep.shape, np.float32)
    for s, (m, b) in enumerate(zip(tokens, budgets)):
        kept = min(m, b)
        assert int(n[s]) == kept
        c, d = int(w.page_offsets[s]) * page, int(offs[s]) * page
        src, to = kvtools.token_rows(w, s), kvtools.token_rows(dst, s, kept)
        for a in range(layers):
            for h in range(kv_heads):
                ww = weights[a, h, c:c + m].numpy()
                idx = kvtools.evict(ww, m, b, sinks, recent)
                want_keep[a, h, d:d + kept], want_left[a, h, d:d + kept] = idx, ww[idx]
                for plane in (2 * a, 2 * a + 1):
                    want[plane, torch.from_numpy(to), h] = before[plane, torch.from_numpy(src[idx]), h]
    assert (keep.cpu().numpy() == want_keep).all()
    assert np.array_equal(left.cpu().numpy(), want_left, equal_nan=True)
    assert (pool.cpu().view(torch.int16) == want.view(torch.int16)).all()
    return w, dst, pool, keep, left, n


@pytest.mark.gpu
@pytest.mark.parametrize("kv_heads,dim,page,sinks,recent", [(2, 64, 16, 0, 0), (1, 128, 8, 4, 20), (3, 8, 7, 1, 29),
                                                            (8, 128, 64, 30, 0), (2, 40, 1, 0, 30)])
def test_evict(cuda_device, kv_heads, dim, page, sinks, recent):
    tokens = [0, 1, 29, 30, 31, 64, 500, 513, 2000, 5]
    budgets = [30, 30, 30, 30, 30, 33, 128, 512, 777, 30]
    evict_case(tokens, budgets, kv_heads=kv_heads, dim=dim, page=page, sinks=sinks, recent=recent, spare=1)


@pytest.mark.gpu
def test_evict_long_sequences(cuda_device):
    evict_case([70001, 20000], [1000, 19999], kv_heads=1, layers=1, dim=8, sinks=4, recent=100)


@pytest.mark.gpu
def test_evict_ties_and_special_weights(cuda_device):
    """Equal weights stay by lower index; -0 equals 0; infinities count as such; NaN goes first."""
    tokens, budgets = [600, 600, 600, 600], [100, 333, 250, 599]
    g = torch.Generator().manual_seed(0)
    weights = torch.randint(0, 3, (1, 2, 4 * 608), generator=g).float()
    weights[0, 0, 608:1216] = 0.0
    weights[0, 0, 608:1216:3] = -0.0
    special = torch.tensor([math.nan, math.inf, -math.inf, 0.0, -0.0, 1e-45, -1e-45, 3e38, -3e38, -1.0])
    weights[0, 1, 1216:] = special[torch.randint(0, 10, (1216,), generator=g)]
    evict_case(tokens, budgets, layers=1, weights=weights)


@pytest.mark.gpu
def test_evict_zero_budget_and_everything_kept(cuda_device):
    evict_case([40, 50, 0], [0, 50, 0])
    evict_case([40, 50], [25, 25], sinks=20, recent=5)   # nothing is left to rank


@pytest.mark.gpu
def test_evict_sequences_shorter_than_what_always_stays(cuda_device):
    """A budget of the whole sequence holds it, also below sinks + recent; the same budget behind it does not."""
    evict_case([2, 5, 0, 43, 44, 700], [2, 5, 0, 43, 43, 100], sinks=7, recent=36)
    evict_case([2, 5, 700], [2, 60, 100], layers=1, sinks=7, recent=36)
    with pytest.raises(Exception, match="below sinks"):
        evict_case([2, 44], [2, 42], sinks=7, recent=36)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [14335, 14336, 14337, 30000])
def test_evict_around_what_shared_memory_holds(cuda_device, n):
    g = torch.Generator().manual_seed(n)
    weights = torch.randint(0, 50, (1, 1, -(-n // 16) * 16), generator=g).float()
    evict_case([n], [4099], kv_heads=1, layers=1, dim=8, sinks=3, recent=17, weights=weights)


@pytest.mark.gpu
def test_evict_reports_bad_tables(cuda_device):
    w, free = kvtools.tables([40, 50], taken=4)
    dst = KvWorkload(w.planes, w.pool_pages, 16, w.token_bytes, np.array([20, 20], np.uint32),
                     np.array([0, 2, 4], np.uint64), free[:4].copy())
    pool = kvtools.make_pool(w, 2, 64, BF16).cuda()
    weights = torch.rand((1, 2, int(w.page_offsets[-1]) * 16), device="cuda")
    for name, change, message in (("page_table", 1, "outside the pool"), ("dst_page_table", 3, "outside the pool"),
                                  ("seq_tokens", 1, "more tokens"), ("budgets", 0, "past the destination")):
        ev = KvEvict(w, dst, 2)
        getattr(ev._tables, name)[change] = 1_000_000
        # every token of sequence 0 is kept or ranked: its first page holds kept ones for certain
        ev.run(pool, torch.ones_like(weights))
        with pytest.raises(_native.TcxError, match=message):
            if name == "page_table":
                getattr(ev._tables, name)[change] = int(w.page_table[change])
            ev.check_status()
    ev = KvEvict(w, dst, 2)
    refused("weights must be", lambda: ev.run(pool, weights[:, :1]))
    refused("weights must be", lambda: ev.run(pool, weights.half()))


@pytest.mark.gpu
def test_evict_with_more_sinks_than_64_bits_hold(cuda_device):
    """Everything stays while the budget holds it; of a sequence that outgrows the budget, its first tokens."""
    w, free = kvtools.tables([20], spare=2, taken=2)
    pool = kvtools.make_pool(w, 2, 64, BF16).cuda()
    dst = KvWorkload(w.planes, w.pool_pages, 16, w.token_bytes, np.array([25], np.uint32), np.array([0, 2], np.uint64),
                     free[:2].copy())
    weights = torch.rand((1, 2, int(w.page_offsets[-1]) * 16), device="cuda")
    for sinks, recent, want in (((1 << 64) + 3, 0, np.arange(25)), (0, (1 << 64) + 3, np.arange(15, 40)),
                                (7, 1 << 64, np.r_[:7, 22:40])):
        ev = KvEvict(w, dst, 2, sinks=sinks, recent=recent)
        assert (ev.run(pool, weights)[0][0, :, :20].cpu().numpy() == np.arange(20)).all()
        ev.seq_tokens.fill_(40)
        assert (ev.run(pool, weights)[0][0, :, :25].cpu().numpy() == want).all()
        ev.check_status()


# ---------------------------------------------------------------- together

@pytest.mark.gpu
def test_decode_with_eviction_as_a_server_runs_it(cuda_device):
    """Prompt, decode steps that accumulate weights, eviction to new pages, more decode steps there, and
    the gather of the shortened sequences, against the same program in 64 bits."""
    kv_heads, group, dim, page, layers = 2, 4, 64, 16, 2
    tokens, budget, steps = [150, 60, 90], 64, 3
    w, free = kvtools.tables(tokens, page, kv_heads, dim, 2 * layers, spare=1, taken=18)
    pool = kvtools.make_pool(w, kv_heads, dim, BF16).cuda()
    weights = torch.zeros((layers, kv_heads, int(w.page_offsets[-1]) * page), device="cuda")
    prompt = KvAttention(w, 8, kv_heads, query_tokens=tokens)
    rng = torch.Generator(device="cuda").manual_seed(3)
    total = np.zeros(0)
    for layer in range(layers):
        q = torch.randn((sum(tokens), 8, dim), generator=rng, device="cuda").to(BF16)
        check(prompt.run(pool, layer, q, weights=weights[layer]),
              kvtools.attention(w, pool, layer, q, tokens), BF16, 150)
    decode = KvAttention(w, 8, kv_heads)
    now = list(tokens)
    for _ in range(steps):
        now = [n + 1 for n in now]
        decode.seq_tokens.add_(1)
        for layer in range(layers):
            q = torch.randn((3, 8, dim), generator=rng, device="cuda").to(BF16)
            ref = kvtools.attention(w, pool, layer, q, [1] * 3, tokens=now)
            check(decode.run(pool, layer, q, weights=weights[layer]), ref, BF16, 160)
    decode.check_status()
    total = weights.sum(-1)  # every query row's weights sum to one
    assert (total - group * (sum(tokens) + 3 * steps)).abs().max() < 1e-3 * float(total.max())
    dst_pages = [6, 6, 6]
    dst = KvWorkload(w.planes, w.pool_pages, page, w.token_bytes, np.full(3, budget, np.uint32),
                     np.concatenate([[0], np.cumsum(dst_pages)]).astype(np.uint64), free[:18].copy())
    ev = KvEvict(w, dst, kv_heads, sinks=2, recent=16)
    ev.seq_tokens.copy_(decode.seq_tokens)
    keep, left, length = ev.run(pool, weights)
    ev.check_status()
    assert length.tolist() == [min(n, budget) for n in now]
    for s, n in enumerate(now):
        c, d = int(w.page_offsets[s]) * page, int(dst.page_offsets[s]) * page
        for a in range(layers):
            for h in range(kv_heads):
                idx = kvtools.evict(weights[a, h, c:c + n].cpu().numpy(), n, budget, 2, 16)
                assert keep[a, h, d:d + len(idx)].tolist() == idx.tolist()
    after = KvAttention(dst, 8, kv_heads)
    after.seq_tokens.copy_(length)
    now = length.tolist()
    for _ in range(steps):
        now = [n + 1 for n in now]
        after.seq_tokens.add_(1)
        for layer in range(layers):
            q = torch.randn((3, 8, dim), generator=rng, device="cuda").to(BF16)
            ref = kvtools.attention(dst, pool, layer, q, [1] * 3, tokens=now)
            check(after.run(pool, layer, q, weights=left[layer]), ref, BF16, 160)
    after.check_status()
    short = KvWorkload(**{**dst.__dict__, "seq_tokens": np.array(now, np.uint32),
                          "page_offsets": dst.page_offsets})
    short.page_offsets = np.concatenate([[0], np.cumsum([-(-n // page) for n in now])]).astype(np.uint64)
    short.page_table = np.concatenate([dst.page_table[int(dst.page_offsets[s]):int(dst.page_offsets[s])
                                                      + -(-n // page)] for s, n in enumerate(now)])
    g = KvGatherHash(short, leaf=4096)
    g.run(pool)
    g.check_status()
    for s, n in enumerate(now):
        rows = torch.from_numpy(kvtools.token_rows(short, s)).cuda()
        assert (g.sequence(s).view(torch.int16) == pool[:, rows].reshape(-1).view(torch.int16)).all()
