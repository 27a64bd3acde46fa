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
from test_gpu_streaming import DEVICE, Cache, evict64, evict_params, paged_params  # noqa: E402


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


@pytest.mark.parametrize("which,at", [(1, 2 ** 25), (1, 2 ** 25 + 4), (2, 2 ** 22), (2, 2 ** 22 + 64), (0, 2 ** 23), (1, 2 ** 24 + 12), (0, 2 ** 27), (2, 2 ** 26 - 4), (0, 2 ** 20 + 40),
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
