"""Streaming attention (gonano_b200/streaming.py) at the calls that its documentation allows and a rollout rarely makes: empty pools
and steps, tables that name their own pages, values that are not finite, gradients of very different sizes.  The float64 statements
and the bounds are those of test_gpu_streaming.py.
"""
import ctypes as C
import math

import pytest

torch = pytest.importorskip("torch")

from gonano_b200 import _lib, streaming  # noqa: E402
from gonano_b200._lib import GonanoError  # noqa: E402
from test_gpu_streaming import DEVICE, FLOOR, PRODUCT, Cache, attend64, check_paged, close, evict64, evict_params, paged_params, score_bound, sink_params, tensors, visible, window_reference  # noqa: E402


@pytest.fixture(scope="module")
def lib():
    from gonano_b200 import build
    build.build()
    return _lib.load()


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


# ---------------------------------------------------------------- pools without pages

@pytest.mark.parametrize("shape", [dict(rows=4, tokens=4, max_query=1), dict(rows=4, tokens=1024, max_query=512), dict(rows=4, tokens=64, max_query=16, mass_out=256)])
def test_workspace_does_not_go_by_the_pages_address(lib, shape):
    """Asked for before the pages are there, it is what the call wants."""
    sizes = []
    for address in (None, 256):
        p = paged_params(n_head=8, n_kv_head=1, head_dim=128, page_size=64, pages=600, table_width=136, max_context=8704, key_pages=address, value_pages=address, **shape)
        n = C.c_int64()
        assert lib.gn_attention_paged_workspace(C.byref(p), C.byref(n)) == 0
        sizes.append(n.value)
    assert sizes[0] == sizes[1]
    # the packed keys and values of a chunk: 4 bytes an element of 4 x 8704 keys and as many values
    assert sizes[0] > (2 * 4 * 8704 * 128 * 4 if shape["max_query"] > 2 else 0)


@pytest.mark.gpu
@pytest.mark.parametrize("count", [1, 3, 40])
def test_a_pool_without_pages(count):
    """No key is there: zeros and -inf, by every kernel."""
    q = torch.randn(2 * count, 8, 64, device=DEVICE)
    pages = torch.zeros(0, 2, 16, 64, device=DEVICE)
    new = torch.randn(2 * count, 2, 64, device=DEVICE)
    out, lse = streaming.paged_attention(q, pages, pages.clone(), torch.zeros(2, 0, dtype=torch.int32, device=DEVICE), ints(0, count, 2 * count), ints(0, 0), count,
                                         new_key=new, new_value=new, out=torch.full_like(q, 3.0))
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())


# ---------------------------------------------------------------- eviction

@pytest.mark.parametrize("over", [dict(budget=2 ** 30 + 1, new_width=2 ** 27), dict(budget=2 ** 31 - 1, new_width=2 ** 28), dict(table_width=2 ** 27, max_context=32),
                                  dict(table_width=2 ** 30 // 16 + 1, max_context=32)])
def test_evict_refuses_more_keys_than_its_indices_count(lib, over):
    """Steps of a block over 2^31 keys would leave 32 bits: refused, whatever the rows."""
    for rows in (0, 2):
        assert lib.gn_cache_evict(C.byref(evict_params(rows=rows, **over)), None, None, None, None) == 1
        assert b"exceeds 2^30" in lib.gn_last_error()
    assert lib.gn_cache_evict(C.byref(evict_params(rows=0, table_width=2 ** 26, new_width=2 ** 26, budget=2 ** 30, max_context=32)), None, None, None, None) == 0


EVICT_BUFFERS = dict(key_pages=2 ** 20, value_pages=2 ** 21, mass=2 ** 22, page_table=2 ** 23, new_table=2 ** 24, context_lens=2 ** 25)   # addresses that are never read
EVICT_OUTPUTS = [2 ** 26, 2 ** 27, 2 ** 28]   # kept, new_lens, mass_out


@pytest.mark.parametrize("which,at", [(1, 2 ** 25 - 4), (1, 2 ** 25 + 4), (2, 2 ** 22), (2, 2 ** 22 + 64), (0, 2 ** 23), (1, 2 ** 24 + 12), (0, 2 ** 27), (2, 2 ** 26 - 4), (0, 2 ** 20 + 40),
                                      (2, 2 ** 21)])
def test_evict_refuses_shared_memory(lib, which, at):
    """Lengths written over the lengths that are read, weights over the weights, and so on: the answer would go by which block came first."""
    outputs = list(EVICT_OUTPUTS)
    outputs[which] = at
    assert lib.gn_cache_evict(C.byref(evict_params(**EVICT_BUFFERS)), *outputs, None) == 1
    assert b"shares memory" in lib.gn_last_error()


@pytest.mark.gpu
def test_evict_buffers_side_by_side(lib):
    """Outputs directly behind one another and behind the lengths that are read are no shared memory."""
    rows, heads, n, budget = 2, 2, 32, 16
    pages = torch.randn(2, 4, heads, 16, 64, device=DEVICE)
    mass = torch.rand(rows, heads, n, device=DEVICE)
    table = ints(0, 1, 2, 3).view(rows, 2)
    room = torch.cat([ints(32, 20), torch.full((rows + rows * heads * budget,), -9, dtype=torch.int32, device=DEVICE)])
    want = streaming.evict_pages(pages[0].clone(), pages[1].clone(), mass, table, ints(32, 20), budget, 1, 2)
    p = evict_params(key_pages=pages[0].data_ptr(), value_pages=pages[1].data_ptr(), mass=mass.data_ptr(), page_table=table.data_ptr(), new_table=table.data_ptr(),
                     context_lens=room.data_ptr())
    assert lib.gn_cache_evict(C.byref(p), room[2 * rows:].data_ptr(), room[rows:].data_ptr(), None, torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(room[rows:2 * rows], want[1]) and torch.equal(room[2 * rows:].view_as(want[0]), want[0])


@pytest.mark.gpu
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("budget", [0, 16, 100, 400])
def test_evict_with_the_lengths_in_one_place(lib, in_place, budget):
    """new_lens over context_lens, as a cache that is compacted in place keeps them: what two arrays give, for every head."""
    lens, heads, page, width = [300, 90, 16, 0, 299], 6, 16, 20
    extra = max(1, -(-budget // page))
    cache = Cache(len(lens), heads, 32, page, width + extra, seed=46)
    cache.fill(lens)
    table, other = cache.table[:, :width].contiguous(), cache.table[:, width:].contiguous()
    target = table if in_place else other
    if in_place and budget > width * page:
        budget = width * page
    mass = torch.rand(len(lens), heads, width * page, generator=cache.gen, device=DEVICE)
    sinks, recent = min(2, budget), min(7, max(0, budget - 2))
    k, v = cache.k.clone(), cache.v.clone()
    want = streaming.evict_pages(k, v, mass, table, ints(*lens), budget, sinks, recent, new_table=target)
    for _ in range(5):
        k2, v2, here = cache.k.clone(), cache.v.clone(), ints(*lens)
        kept = torch.full((len(lens), heads, max(1, budget)), -9, dtype=torch.int32, device=DEVICE)
        p = evict_params(rows=len(lens), n_kv_head=heads, head_dim=32, page_size=page, pages=k2.shape[0], table_width=width, new_width=target.shape[1], mass_stride=width * page,
                         max_context=width * page, budget=budget, sinks=sinks, recent=recent, key_pages=k2.data_ptr(), value_pages=v2.data_ptr(), mass=mass.data_ptr(),
                         page_table=table.data_ptr(), new_table=target.data_ptr(), context_lens=here.data_ptr())
        assert lib.gn_cache_evict(C.byref(p), kept.data_ptr(), here.data_ptr(), None, torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(here, want[1]) and (budget == 0 or torch.equal(kept, want[0]))
        assert torch.equal(k2.nan_to_num(9.0), k.nan_to_num(9.0)) and torch.equal(v2.nan_to_num(9.0), v.nan_to_num(9.0))


@pytest.mark.gpu
@pytest.mark.parametrize("dim,page", [(128, 64), (64, 16), (33, 1), (80, 7)])
@pytest.mark.parametrize("mixed", [False, True])
def test_evict_to_a_copy_of_the_own_pages(dim, page, mixed):
    """new_table a narrower copy of page_table: in place, though it is another tensor.  Mixed: every second page is a fresh one."""
    lens, heads, budget, sinks, recent = [1300, 900, 500, 20, 0], 2, 600, 3, 100
    width, kept_pages = -(-1300 // page), -(-budget // page)
    cache = Cache(len(lens), heads, dim, page, width + kept_pages, seed=30)
    cache.fill(lens)
    table, target = cache.table[:, :width].contiguous(), cache.table[:, :kept_pages].contiguous()
    if mixed:
        target[:, 1::2] = cache.table[:, width:width + kept_pages][:, 1::2]
    mass = torch.rand(len(lens), heads, width * page, generator=cache.gen, device=DEVICE)
    want = evict64(mass.cpu(), lens, budget, sinks, recent)
    for _ in range(5):   # an order left to chance shows in some of the calls
        k, v = cache.k.clone(), cache.v.clone()
        kept, new_lens, _ = streaming.evict_pages(k, v, mass, table, ints(*lens), budget, sinks, recent, new_table=target)
        assert new_lens.tolist() == [min(n, budget) for n in lens]
        touched = torch.zeros(k.shape[:3], dtype=torch.bool, device=DEVICE)
        for r in range(len(lens)):
            for h in range(heads):
                w = torch.tensor(want[r * heads + h], dtype=torch.long, device=DEVICE)
                assert torch.equal(kept[r, h, :len(w)].long(), w)
                slots = torch.arange(len(w), device=DEVICE)
                src, dst = table[r].long()[w // page], target[r].long()[slots // page]
                touched[dst, h, slots % page] = True
                for now, then in ((k, cache.k), (v, cache.v)):
                    assert torch.equal(now[dst, h, slots % page], then[src, h, w % page])
        for now, then in ((k, cache.k), (v, cache.v)):
            assert torch.equal(now[~touched].nan_to_num(9.0), then[~touched].nan_to_num(9.0))


# ---------------------------------------------------------------- weights

@pytest.mark.gpu
@pytest.mark.parametrize("tokens,max_query", [(0, 4), (3, 0), (0, 0), (2, 1)])
@pytest.mark.parametrize("start", ["mass", "nothing", "one buffer", "a copy"])
def test_weights_of_a_step_without_tokens(tokens, max_query, start):
    """No row has a new token: mass_out holds what mass holds (0 where there is none) up to every row's length, and is left as it is behind."""
    lens, heads, page, width = [40, 0, 300, 512, 600], 2, 32, 16
    cache = Cache(len(lens), heads, 64, page, width, seed=31)
    mass = torch.rand(len(lens), heads, width * page, generator=cache.gen, device=DEVICE)
    before, out = mass.clone(), torch.full_like(mass, 7.0)
    q = torch.randn(tokens, 4, 64, device=DEVICE)
    got = streaming.paged_attention(q, cache.k, cache.v, cache.table, ints(*[0] * (len(lens) + 1)), ints(*lens), max_query, scale=0.125,
                                    mass=None if start == "nothing" else mass, mass_out={"one buffer": mass, "a copy": None}.get(start, out))[2]
    assert torch.equal(mass, before)
    for r, n in enumerate(lens):
        assert torch.equal(got[r, :, :n], before[r, :, :n] * (0.0 if start == "nothing" else 1.0))
        assert torch.equal(got[r, :, n:], (before if start in ("one buffer", "a copy") else torch.full_like(mass, 7.0))[r, :, n:])


def test_weights_of_a_step_without_tokens_want_the_lengths(lib):
    view = _lib.GnView(None, 64, 64, 64)
    assert lib.gn_attention_paged(C.byref(paged_params(tokens=0, mass_out=2 ** 20)), C.byref(view), None, None, 0, None) == 1
    assert b"context_lens" in lib.gn_last_error()
    assert lib.gn_attention_paged(C.byref(paged_params(tokens=0, mass_out=2 ** 20, max_context=0)), C.byref(view), None, None, 0, None) == 0


@pytest.mark.parametrize("shift", [4, 64, 2 * 2 * 32 * 4 - 4, -4, -256])
def test_weights_that_share_a_part_are_refused(lib, shift):
    n, view = C.c_int64(), _lib.GnView(None, 64, 64, 64)
    p = paged_params(mass=2 ** 20, mass_out=2 ** 20 + shift)
    assert lib.gn_attention_paged(C.byref(p), C.byref(view), None, None, 0, None) == 1 and b"share a part" in lib.gn_last_error()
    assert lib.gn_attention_paged_workspace(C.byref(p), C.byref(n)) == 0   # goes by no address
    for apart in (0, 2 * 2 * 32 * 4, -2 * 2 * 32 * 4):
        p = paged_params(mass=2 ** 20, mass_out=2 ** 20 + apart)
        assert lib.gn_attention_paged(C.byref(p), C.byref(view), None, None, 0, None) == 1 and b"share a part" not in lib.gn_last_error()


# ---------------------------------------------------------------- numbers

@pytest.mark.parametrize("big", [2 ** 31, 2 ** 32, 2 ** 32 + 3, -2 ** 31 - 1, 2 ** 70])
def test_numbers_beyond_32_bits_are_refused(big):
    """2^32 sinks are not 0 sinks."""
    x, table, lens = torch.zeros(1, 2, 4, 8), torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for name in ("sinks", "window"):
        with pytest.raises(GonanoError, match=f"{name}: {big} is outside"):
            streaming.sink_attention_forward(x, x, x, **{"sinks": 0, "window": -1, name: big})
        with pytest.raises(GonanoError, match=f"{name}: {big} is outside"):
            streaming.sink_attention_backward(x, x, x, x, x, x[..., 0], **{"sinks": 0, "window": -1, name: big})
    for name in ("max_query", "max_context", "sinks", "window"):
        with pytest.raises(GonanoError, match=f"{name}: {big} is outside"):
            streaming.paged_attention(x[0], x, x, table, lens, lens, **{"max_query": 1, name: big})
    for name in ("budget", "sinks", "recent", "max_context"):
        with pytest.raises(GonanoError, match=f"{name}: {big} is outside"):
            streaming.evict_pages(x, x, x[0], table, lens, **{"budget": 1, name: big})


# ---------------------------------------------------------------- values that are not finite, rows shorter than their tokens, missing pages

CLEAN = 2.0 ** -16   # between two passes that differ in other queries' operands only: twice the rounding of each, as in test_gpu_streaming.py


@pytest.mark.gpu
@pytest.mark.parametrize("count,heads,kv_heads", [(1, 4, 2), (12, 2, 2), (12, 1, 1), (40, 4, 2), (140, 2, 1)])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("old", [False, True])
def test_non_finite_in_the_cache(count, heads, kv_heads, value, which, old):
    """A cached key or value (or a new token's) that is not finite reaches only the queries that see it, and the weights of the keys that those see."""
    n, page, window, sinks, dim = 300, 16, 4, 2, 64
    at = n - count - 3 if old else n - (count + 1) // 2
    cache = Cache(2, kv_heads, dim, page, -(-n // page), seed=32)
    cache.fill([n - count, n - count])
    q = torch.randn(2 * count, heads, dim, generator=cache.gen, device=DEVICE)
    new = [torch.randn(2 * count, kv_heads, dim, generator=cache.gen, device=DEVICE) for _ in range(2)]
    got = []
    for bad in (False, True):
        k, v, nk, nv = cache.k.clone(), cache.v.clone(), *(x.clone() for x in new)
        if bad:
            if old:
                (k if which == "k" else v)[int(cache.table[0, at // page]), :, at % page, 3] = value
            else:
                (nk if which == "k" else nv)[at - (n - count), :, 3] = value
        got.append(streaming.paged_attention(q, k, v, cache.table, ints(0, count, 2 * count), ints(n, n), count, new_key=nk, new_value=nv, sinks=sinks, window=window,
                                             scale=0.125, mass_out=torch.zeros(2, kv_heads, cache.table.shape[1] * page, device=DEVICE)))
    pos, keys = torch.arange(n - count, n, device=DEVICE), torch.arange(n, device=DEVICE)
    see = visible(pos, keys, window, sinks)
    hit = torch.zeros(2 * count, dtype=torch.bool, device=DEVICE)
    hit[:count] = see[:, at]
    (clean, clean_lse, clean_mass), (out, lse, mass) = got
    assert bool(hit.any())
    if which == "v" or math.isnan(value):
        assert not bool(out[hit][..., 3].isfinite().any())
    close(out[~hit], clean[~hit].double(), CLEAN, "out")
    close(lse[~hit], clean_lse[~hit].double(), CLEAN, "lse")
    reached = see[hit[:count]].any(0)
    close(mass[0, :, :n][:, ~reached], clean_mass[0, :, :n][:, ~reached].double(), CLEAN, "mass")
    close(mass[1], clean_mass[1].double(), CLEAN, "mass of the other row")


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["q", "k", "v", "dout"])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("heads,dim", [(1, 64), (4, 128)])
def test_non_finite_in_a_training_pass(which, value, heads, dim):
    """It reaches the gradients of the queries that see the key (or hold the value themselves) and of the keys that those see, no others."""
    T, window, sinks, at = 700, 20, 2, 350
    clean = tensors(1, heads, 1, T, dim, seed=33)
    bad = [x.clone() for x in clean]
    bad[("q", "k", "v", "dout").index(which)][0, 0, at, 3] = value
    results = []
    for q, k, v, dout in (clean, bad):
        out, lse = streaming.sink_attention_forward(q, k, v, sinks, window, 0.1)
        results.append((out, lse, *streaming.sink_attention_backward(q, k, v, out, dout, lse, sinks, window, 0.1)))
    i = torch.arange(T, device=DEVICE)
    see = visible(i, i, window, sinks)
    queries = see[:, at] if which in ("k", "v") else i == at
    keys = see[queries].any(0)
    rows = torch.zeros(heads, T, dtype=torch.bool, device=DEVICE)
    rows[:heads if which in ("k", "v") else 1] = queries
    (out, lse, dq, dk, dv), (out2, lse2, dq2, dk2, dv2) = results
    fine = ~rows if which != "dout" else torch.ones_like(rows)
    # sums of up to 21 x heads terms of size 1 and the largest sinks' of T x heads: relative to the clean tensors' largest
    for name, a, b, where in (("out", out[0], out2[0], fine), ("lse", lse[0], lse2[0], fine), ("dq", dq[0], dq2[0], ~rows), ("dk", dk[0, 0], dk2[0, 0], ~keys), ("dv", dv[0, 0], dv2[0, 0], ~keys)):
        close(b[where], a[where].double(), CLEAN * max(1.0, float(a[a.isfinite()].abs().max())), name)
    if math.isnan(value):
        assert not bool(dq2[0][rows].isfinite().any())
        if which in ("q", "dout"):
            assert not bool(dk2[0, 0][keys].isfinite().any())


@pytest.mark.gpu
@pytest.mark.parametrize("counts,lens,heads,kv_heads,dim,page,window,sinks", [
    ([1, 0, 1, 1], [300, 20, 0, 5], 4, 2, 40, 8, 20, 4),
    ([7, 9], [2000, 3], 2, 2, 128, 256, 30, 900),
    ([5, 4, 8, 2], [3, 0, 8, 1], 2, 1, 64, 16, -1, 0),
    ([16, 1], [9, 1], 1, 1, 128, 4, 3, 1),
    ([40, 30, 12], [17, 0, 200], 4, 2, 64, 16, -1, 0),
    ([300, 200], [150, 1999], 2, 1, 80, 24, 50, 700),
])
def test_rows_shorter_than_their_new_tokens(counts, lens, heads, kv_heads, dim, page, window, sinks):
    """The first tokens then stand before the cache: they see nothing and are not written; sinks beyond most of a long row."""
    rows, group, scale = len(counts), heads // kv_heads, 1 / math.sqrt(dim)
    cache = Cache(rows, kv_heads, dim, page, max(1, -(-max(lens) // page)), seed=34)
    cache.fill([max(0, n - c) for n, c in zip(lens, counts)])
    tokens = sum(counts)
    q = torch.randn(tokens, heads, dim, generator=cache.gen, device=DEVICE)
    nk, nv = (torch.randn(tokens, kv_heads, dim, generator=cache.gen, device=DEVICE) for _ in range(2))
    old = cache.k.clone()
    starts = [sum(counts[:r]) for r in range(rows + 1)]
    before = torch.rand(rows, kv_heads, cache.table.shape[1] * page, generator=cache.gen, device=DEVICE)
    out, lse, mass = streaming.paged_attention(q, cache.k, cache.v, cache.table, ints(*starts), ints(*lens), max(counts), new_key=nk, new_value=nv, sinks=sinks,
                                               window=window, scale=scale, mass=before)
    written = torch.zeros(old.shape[:3], dtype=torch.bool, device=DEVICE)
    for r, (c, n) in enumerate(zip(counts, lens)):
        b, new = starts[r], min(c, n)
        k64, v64 = cache.row(r, n)
        assert torch.equal(k64[n - new:], nk[b + c - new:b + c].double()) and torch.equal(v64[n - new:], nv[b + c - new:b + c].double())
        for j in range(n - new, n):
            written[int(cache.table[r, j // page]), :, j % page] = True
        see = visible(torch.arange(n - c, n, device=DEVICE), torch.arange(n, device=DEVICE), window, sinks)
        for h in range(kv_heads):
            mine = slice(h * group, (h + 1) * group)
            qq = q[b:b + c, mine].double().transpose(0, 1)
            o, l, w = attend64(qq, k64[:, h], v64[:, h], see, scale)
            e = (2 * score_bound(qq, k64[:, h], scale) if qq.numel() else 0.0) + PRODUCT
            close(out[b:b + c, mine].transpose(0, 1), o, e * torch.einsum("gnm,md->gnd", w, v64[:, h].abs()) + FLOOR * (n + 2) * float(v64.abs().max() if n else 0), f"out of row {r}")
            close(lse[b:b + c, mine].transpose(0, 1), l, e * (1 + l.abs()), f"lse of row {r}")
            want = w.sum((0, 1))
            want[:max(0, n - c)] += before[r, h, :max(0, n - c)].double()
            close(mass[r, h, :n], want, e * want + 2.0 ** -22 * want, f"mass of row {r}")
            assert torch.equal(mass[r, :, n:], before[r, :, n:])
    assert torch.equal(cache.k[~written].nan_to_num(9.0), old[~written].nan_to_num(9.0))


@pytest.mark.gpu
@pytest.mark.parametrize("counts,group", [([1, 1], 2), ([6, 3], 2), ([6, 3], 1), ([90, 33], 2)])
@pytest.mark.parametrize("window,sinks", [(-1, 0), (60, 5)])
def test_new_tokens_without_a_page(counts, group, window, sinks):
    """A new token whose slot lies on a page that does not exist is neither written nor seen, its neighbours are."""
    check_paged(counts, [400, 333], 2 * group, 2, 64, 32, window, sinks, hide=(0, 12))
    check_paged(counts, [385, 353], 2 * group, 2, 64, 32, window, sinks, hide=(0, 12))
    check_paged(counts, [400, 353], 2 * group, 2, 64, 32, window, sinks, hide=(1, 11))


# ---------------------------------------------------------------- gradients of quiet tokens

def norm_error(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.gpu
@pytest.mark.parametrize("ratio", [1.0, 1e-3, 1e-5, 1e-7])
@pytest.mark.parametrize("heads,kv_heads,T,window,sinks,begin,end", [
    (1, 1, 768, 512, 4, 300, 556),      # a stretch in the middle
    (8, 1, 900, 512, 4, 301, 557),      # the heads of a group side by side
    (6, 2, 900, 32, 0, 200, 456),       # keys that only quiet tokens see
    (1, 1, 700, -1, 0, 444, 700),       # at the end, under a causal mask: again such keys
    (2, 1, 2100, 100, 2, 1000, 1256),
])
def test_gradients_of_quiet_tokens(ratio, heads, kv_heads, T, window, sinks, begin, end):
    """256 tokens whose dO is a small part of the others': their dQ, dK and dV are as precise as float32, relative to their own norm.

    2e-6: operands of 22 bits, float32 sums and an exponential make 3e-7 to 9e-7 of the norm where all tokens are alike, in float32 too."""
    q, k, v, dout = tensors(1, heads, kv_heads, T, 128, seed=40)
    dout[:, :, begin:end] *= ratio
    scale = 128 ** -0.5
    out, lse = streaming.sink_attention_forward(q, k, v, sinks, window, scale)
    got = dict(zip(("dq", "dk", "dv"), streaming.sink_attention_backward(q, k, v, out, dout, lse, sinks, window, scale)))
    want, _ = window_reference(q, k, v, dout, None, window, sinks, scale)
    errors = {n: (norm_error(g[:, :, begin:end], want[n][:, :, begin:end]), norm_error(g, want[n])) for n, g in got.items()}
    print(ratio, errors)
    assert all(e < 2e-6 for pair in errors.values() for e in pair), errors


@pytest.mark.gpu
def test_gradients_of_tokens_and_heads_of_every_size():
    """dO of every token and head at its own power of ten, zeros and whole tiles of zeros among them: every row of dQ is precise."""
    T, heads = 500, 4
    q, k, v, dout = tensors(2, heads, 1, T, 64, seed=41)
    gen = torch.Generator(device=DEVICE).manual_seed(42)
    size = 10.0 ** torch.randint(-9, 1, (2, heads, T, 1), generator=gen, device=DEVICE).float()
    size[:, :, ::17], size[0, :, 64:200], size[1, 2] = 0.0, 0.0, 1e-12
    dout = dout * size
    out, lse = streaming.sink_attention_forward(q, k, v, 3, 60, 0.125)
    dq, dk, dv = streaming.sink_attention_backward(q, k, v, out, dout, lse, 3, 60, 0.125)
    want, _ = window_reference(q, k, v, dout, None, 60, 3, 0.125)
    assert bool((dq[(size == 0).expand_as(dq)] == 0).all())
    rows = (dq.double() - want["dq"]).norm(dim=-1) / want["dq"].norm(dim=-1)
    rows = rows[(size > 0).squeeze(-1) & (torch.arange(T, device=DEVICE) > 0)]   # the first token sees itself alone: its dQ is 0 but for roundings
    # a component of dO is off by up to 2^-39 2^-6 of the tile's largest: 2^-45 10^12 / 1 = 0.03 for the quietest, 3e-5 at 10^-9 and below 1e-6 from 10^-7 on
    quiet = size[(size > 0) & (torch.arange(T, device=DEVICE) > 0)[None, None, :, None]] < 2e-8
    assert float(rows[~quiet].max()) < 1e-4 and float(rows[~quiet].median()) < 2e-6, (float(rows[~quiet].max()), float(rows[~quiet].median()))
    for name, g in (("dk", dk), ("dv", dv)):
        assert norm_error(g, want[name]) < 2e-6


# ---------------------------------------------------------------- outputs in one place

def test_outputs_that_share_memory_are_refused(lib):
    """The same tensor as two gradients, or attention written over its own inputs."""
    def view(at, heads):
        return _lib.GnView(at, heads * 512, 512, 64)
    p = sink_params(query=view(2 ** 20, 4), key=view(2 ** 21, 2), value=view(2 ** 22, 2))
    at = [2 ** 23, 2 ** 24, 2 ** 25]
    for i, j in ((0, 1), (0, 2), (1, 2)):
        same = list(at)
        same[j] = same[i]
        grads = [view(same[0], 4), view(same[1], 2), view(same[2], 2)]
        assert lib.gn_attention_sink_backward(C.byref(p), C.byref(view(2 ** 26, 4)), C.byref(view(2 ** 27, 4)), 2 ** 28, *map(C.byref, grads), 0, 2 ** 29, 2 ** 30, None) == 1
        assert b"two gradients share memory" in lib.gn_last_error()
    def token_view(at, heads):
        return _lib.GnView(at, 0, 64, heads * 64)
    fields = dict(query=token_view(2 ** 20, 4), new_key=token_view(2 ** 21, 2), new_value=token_view(2 ** 22, 2), key_pages=2 ** 23, value_pages=2 ** 24, page_table=2 ** 25,
                  query_starts=2 ** 26, context_lens=2 ** 27, mass_out=2 ** 19)
    for start in (2 ** 20, 2 ** 21, 2 ** 22):
        assert lib.gn_attention_paged(C.byref(paged_params(**fields)), C.byref(token_view(start, 4)), 2 ** 28, 2 ** 29, 2 ** 20, None) == 1
        assert b"out shares memory" in lib.gn_last_error()


@pytest.mark.gpu
def test_gradients_in_one_tensor_are_refused():
    q, k, v, dout = tensors(1, 2, 2, 16, 32, seed=43)
    out, lse = streaming.sink_attention_forward(q, k, v, 0, -1)
    dq, dk = torch.zeros_like(q), torch.zeros_like(k)
    with pytest.raises(GonanoError, match="two gradients"):
        streaming.sink_attention_backward(q, k, v, out, dout, lse, 0, -1, dq=dq, dk=dk, dv=dk)
    fused = torch.zeros(1, 16, 6, 32, device=DEVICE).transpose(1, 2)   # side by side in one buffer is fine
    want = streaming.sink_attention_backward(q, k, v, out, dout, lse, 0, -1)
    got = streaming.sink_attention_backward(q, k, v, out, dout, lse, 0, -1, dq=fused[:, :2], dk=fused[:, 2:4], dv=fused[:, 4:])
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("a,b,c", [(0, 0, 40), (0, 0, -60), (35, 0, 0), (-35, 0, 0), (0, 50, -30), (0, -50, 60), (20, 30, 10)])
@pytest.mark.parametrize("heads,kv_heads,T,D", [(4, 2, 300, 64), (6, 1, 200, 128)])
def test_powers_of_two_go_through(a, b, c, heads, kv_heads, T, D):
    """Queries times 2^a and keys over 2^a, values times 2^b, dO times 2^c: the same bits, times the powers that the formulas give."""
    q, k, v, dout = tensors(2, heads, kv_heads, T, D, seed=47)
    dout[:, :, 50:90] *= 1e-4
    mask = dict(sinks=3, window=40, scale=0.11)

    def run(q, k, v, dout):
        out, lse = streaming.sink_attention_forward(q, k, v, **mask)
        return out, lse, *streaming.sink_attention_backward(q, k, v, out, dout, lse, **mask)
    plain = run(q, k, v, dout)
    moved = run(q * 2.0 ** a, k * 2.0 ** -a, v * 2.0 ** b, dout * 2.0 ** c)
    for name, x, y, power in zip(("out", "lse", "dq", "dk", "dv"), plain, moved, (b, 0, b + c - a, b + c + a, c)):
        assert torch.equal(y, x * 2.0 ** power), name


# ---------------------------------------------------------------- tiles that arrive late

def cold_calls(call, times):
    """Outputs of the first call, after others on caches filled with something else gave the same bits."""
    room = torch.empty(256 << 20, dtype=torch.uint8, device=DEVICE)
    first, differ = [x.clone() for x in call()], []
    for i in range(times):
        room.fill_(i & 127)
        differ.append(torch.stack([(x != y).sum() for x, y in zip(call(), first)]))
    assert int(torch.stack(differ).sum()) == 0
    return first


@pytest.mark.gpu
@pytest.mark.parametrize("rows,chunk,context,heads,dim,page", [(44, 30, 5246, 4, 96, 256), (12, 64, 8704, 8, 128, 64), (90, 24, 3000, 4, 64, 64)])
def test_long_rows_from_cold_caches(rows, chunk, context, heads, dim, page):
    """Caches larger than L2: key tiles come from memory, more slowly than they are multiplied.  A tile used before it is there shows in the result
    (and ended calls in a device error: its place was handed out twice)."""
    host = torch.Generator().manual_seed(77)
    counts = torch.randint(0, chunk + 1, (rows,), generator=host)
    counts[0], counts[1] = chunk, 0
    lens = torch.randint(context // 2, context + 1, (rows,), generator=host)
    lens[0] = context
    width = -(-context // page)
    gen = torch.Generator(device=DEVICE).manual_seed(44)
    k = torch.randn(rows * width, 1, page, dim, generator=gen, device=DEVICE)
    v = torch.randn(rows * width, 1, page, dim, generator=gen, device=DEVICE)
    table = torch.randperm(rows * width, generator=host).to(torch.int32).view(rows, width).to(DEVICE)
    starts = [int(counts[:r].sum()) for r in range(rows + 1)]
    q = torch.randn(starts[-1], heads, dim, generator=gen, device=DEVICE)
    scale = dim ** -0.5
    out, lse = cold_calls(lambda: streaming.paged_attention(q, k, v, table, ints(*starts), ints(*lens.tolist()), chunk, scale=scale), 60)
    for r in (0, 2, rows - 1):
        b, e, n = starts[r], starts[r + 1], int(lens[r])
        k64, v64 = (x[table[r].long()].reshape(-1, dim)[:n].double() for x in (k, v))
        see = visible(torch.arange(n - (e - b), n, device=DEVICE), torch.arange(n, device=DEVICE), -1, 0)
        qq = q[b:e].double().transpose(0, 1)
        o, l, w = attend64(qq, k64, v64, see, scale)
        if e > b:
            bound = 2 * score_bound(qq, k64, scale) + PRODUCT
            close(out[b:e].transpose(0, 1), o, bound * torch.einsum("gnm,md->gnd", w, v64.abs()) + FLOOR * (n + 2) * float(v64.abs().max()), f"out of row {r}")
            close(lse[b:e].transpose(0, 1), l, bound * (1 + l.abs()), f"lse of row {r}")


@pytest.mark.gpu
@pytest.mark.parametrize("B,H,Hkv,T,D,window,sinks", [(64, 2, 2, 2000, 128, 256, 4), (200, 2, 2, 600, 128, 0, 0), (3, 4, 4, 6000, 128, -1, 0)])
def test_prefill_from_cold_caches(B, H, Hkv, T, D, window, sinks):
    """The same of padded batches: items of a few key tiles, of a single one, of many."""
    q, k, v, _ = tensors(B, H, Hkv, T, D, seed=45)
    out, lse = cold_calls(lambda: streaming.sink_attention_forward(q, k, v, sinks, window, 0.09), 40)
    at = torch.arange(T, device=DEVICE)
    for b in (0, B - 1):
        qq, kk, vv = q[b, :1].double(), k[b, 0].double(), v[b, 0].double()
        o, l, w = attend64(qq, kk, vv, visible(at, at, window, sinks), 0.09)
        bound = 2 * score_bound(qq, kk, 0.09) + PRODUCT
        close(out[b, :1], o, bound * torch.einsum("gnm,md->gnd", w, vv.abs()) + FLOOR * (T + 2) * float(vv.abs().max()), "out")
        close(lse[b, :1], l, bound * (1 + l.abs()), "lse")
