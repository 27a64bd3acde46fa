"""Streaming attention (gonano_b200/streaming.py) against float64 statements of the formulas, its refusals, and its pieces run together.

Tolerances.  A score is a product of head_dim terms: operands kept to 22 bits, terms and sums in float32, which bounds its error by
e = 2^-19 |scale| |q| |k| (22-bit operands 2 * 2^-22, the product of the parts below 22 bits 2^-22, at most 24 roundings of a
partial sum 24 * 2^-24, together below 2^-19).  A weight is then off by at most 2 e relative (numerator and sum), an output by
(2 e + 2^-18) sum p |v| with the same 2^-18 > 2^-19 + 2^-20 for its own product and the sum of the weights.  Gradients propagate
these bounds term by term in `window_reference`.  The largest possible errors add up; measured ones are far below.

Operands that go through f16 pairs (high and low part of a scaled value) have, beside the relative bound, a smallest step: f16's
is 2^-24, so a pair is off by up to 2^-25.  A weight is held as 2^15 p: off by up to FLOOR = 2^-40, whatever p.  A tensor's entry is held
times a power of two that brings its sequence's largest to 2^14 or more: off by up to 2^-39 of the largest.  dS is held times
2^(14 - e), max|dO| max|V| < 2^e <= 2 max|dO| max|V|: off by up to 2^-25 2^(e - 14) <= 2^-38 max|dO| max|V|.
"""
import itertools
import math

import pytest

torch = pytest.importorskip("torch")

from gonano_b200 import _lib, streaming  # noqa: E402
from gonano_b200._lib import GonanoError  # noqa: E402

PRODUCT = 2.0 ** -18
FLOOR = 2.0 ** -40
DEVICE = "cuda"


def visible(positions, keys, window, sinks):
    i, j = positions[:, None], keys[None, :]
    return (j <= i) & ((i - j <= window) | (j < sinks) if window >= 0 else torch.ones_like(j, dtype=torch.bool))


def attend64(q, k, v, see, scale):
    """q [g, n, d], k / v [m, d], see [n, m] in float64: out, lse, weights; what is not seen is not touched."""
    scores = torch.einsum("gnd,md->gnm", q, k) * scale
    scores = torch.where(see, scores, -math.inf)
    top = scores.amax(-1, keepdim=True) if k.shape[0] else torch.full((*scores.shape[:2], 1), -math.inf, dtype=q.dtype, device=q.device)
    top = torch.where(top == -math.inf, 0.0, top)
    w = (scores - top).exp()
    total = w.sum(-1, keepdim=True)
    lse = (top + total.log()).squeeze(-1)
    w = torch.where(total > 0, w / total, 0.0)
    return torch.einsum("gnm,md->gnd", w, v), lse, w


def score_bound(q, k, scale):
    if not k.numel():
        return 0.0
    return 2.0 ** -19 * abs(scale) * float(q.norm(dim=-1).max()) * float(k.norm(dim=-1).max())


def close(got, want, bound, what):
    assert got.dtype == torch.float32
    got = got.double()
    same = (got == want) | ((got - want).abs() <= bound)   # infinities are equal or wrong
    assert bool(same.all()), f"{what}: off by {float((got - want).abs().nan_to_num(math.inf).max()):.3g} where {float(torch.as_tensor(bound).max()):.3g} is allowed"


def window_reference(q, k, v, dout, lengths, window, sinks, scale):
    """Outputs, gradients and their bounds for [B, H, T, D] tensors, one (sequence, kv head) at a time in float64."""
    B, H, T, D = q.shape
    Hkv = k.shape[1]
    g = H // Hkv
    q, k, v, dout = (x.double() for x in (q, k, v, dout))
    res = {n: torch.zeros_like(x) for n, x in (("out", q), ("dq", q), ("dk", k), ("dv", v))}
    res["lse"] = torch.full((B, H, T), -math.inf, dtype=torch.float64, device=q.device)
    bounds = {n: torch.zeros_like(x) for n, x in res.items()}
    for b, h in itertools.product(range(B), range(Hkv)):
        n = T if lengths is None else int(lengths[b].clamp(0, T))
        if n == 0:
            continue
        mine = slice(h * g, (h + 1) * g)
        qq, kk, vv, do = q[b, mine, :n], k[b, h, :n], v[b, h, :n], dout[b, mine, :n]
        at = torch.arange(n, device=q.device)
        see = visible(at, at, window, sinks)
        out, lse, w = attend64(qq, kk, vv, see, scale)
        dp = torch.einsum("gnd,md->gnm", do, vv) - (do * out).sum(-1, keepdim=True)
        ds = w * dp
        res["out"][b, mine, :n], res["lse"][b, mine, :n] = out, lse
        res["dq"][b, mine, :n] = scale * torch.einsum("gnm,md->gnd", ds, kk)
        res["dk"][b, h, :n] = scale * torch.einsum("gnm,gnd->md", ds, qq)
        res["dv"][b, h, :n] = torch.einsum("gnm,gnd->md", w, do)
        e = 2 * score_bound(qq, kk, scale)
        big = [float(x.abs().max()) for x in (qq, kk, vv, do)]
        seen = see.double().expand(w.shape)
        bounds["out"][b, mine, :n] = (e + PRODUCT) * torch.einsum("gnm,md->gnd", w, vv.abs()) + FLOOR * (torch.einsum("gnm,md->gnd", seen, vv.abs()) + 2 * big[2])
        bounds["lse"][b, mine, :n] = (e + PRODUCT) * (1 + lse.abs())
        # ds: the weight's error, and that of dO.v - dO.o (a product each, and the error of o)
        reach = do.norm(dim=-1, keepdim=True) * float(vv.norm(dim=-1).max())
        eds = w * (e * dp.abs() + (e + 2 * PRODUCT) * reach) + PRODUCT * ds.abs() + seen * (FLOOR * dp.abs() + 4 * FLOOR * float(reach.max()))
        bounds["dq"][b, mine, :n] = abs(scale) * torch.einsum("gnm,md->gnd", eds, kk.abs()) + abs(scale) * 2 * FLOOR * big[1] * ds.abs().sum(-1, keepdim=True)
        bounds["dk"][b, h, :n] = abs(scale) * torch.einsum("gnm,gnd->md", eds, qq.abs()) + abs(scale) * 2 * FLOOR * big[0] * ds.abs().sum((0, 1))[:, None]
        bounds["dv"][b, h, :n] = (e + PRODUCT) * torch.einsum("gnm,gnd->md", w, do.abs()) + FLOOR * torch.einsum("gnm,gnd->md", seen, do.abs()) \
            + 2 * FLOOR * big[3] * w.sum((0, 1))[:, None]
    return res, bounds


def tensors(B, H, Hkv, T, D, seed=0, token_major=False):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)

    def make(heads):
        if token_major:   # heads side by side inside a token, with room between tokens
            return torch.randn(B, T, heads + 1, D, generator=gen, device=DEVICE)[:, :, :heads].transpose(1, 2)
        return torch.randn(B, heads, T, D, generator=gen, device=DEVICE)
    return make(H), make(Hkv), make(Hkv), make(H)


def check_window(q, k, v, dout, lengths, window, sinks, scale):
    mask = dict(sinks=sinks, window=window, scale=scale, lengths=lengths)
    out, lse = streaming.sink_attention_forward(q, k, v, **mask)
    dq, dk, dv = streaming.sink_attention_backward(q, k, v, out, dout, lse, **mask)
    want, bounds = window_reference(q, k, v, dout, lengths, window, sinks, scale)
    for name, got in (("out", out), ("lse", lse), ("dq", dq), ("dk", dk), ("dv", dv)):
        close(got, want[name], bounds[name], name)
    return out, lse, dq, dk, dv


SHAPES = [(1, 1, 1, 1, 1), (2, 2, 1, 63, 64), (1, 6, 2, 130, 128), (2, 3, 1, 257, 80), (1, 8, 1, 200, 128), (1, 4, 4, 129, 33), (2, 5, 5, 17, 16), (1, 16, 1, 700, 64)]
MASKS = [(-1, 0), (0, 0), (0, 1), (16, 4), (64, 70), (100, 300), (5000, 3), (127, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("window,sinks", MASKS)
def test_window_and_sinks(shape, window, sinks):
    check_window(*tensors(*shape), None, window, sinks, 1 / math.sqrt(shape[-1]))


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1.0, -0.3, 0.0])
def test_scale(scale):
    check_window(*tensors(1, 4, 2, 150, 64, seed=1), None, 40, 2, scale)


@pytest.mark.gpu
@pytest.mark.parametrize("T,window,sinks", [(300, 60, 5), (129, -1, 0)])
def test_lengths_and_padding(T, window, sinks):
    """Sequences of no, one and all tokens; padding is NaN and infinity and must not be read; lengths outside [0, T] are cut."""
    q, k, v, dout = tensors(6, 4, 2, T, 64, seed=2)
    lengths = torch.tensor([0, 1, T, T + 9, -3, T // 2 + 1], dtype=torch.int32, device=DEVICE)
    for b, n in enumerate(lengths.clamp(0, T).tolist()):
        for x in (q, k, v, dout):
            x[b, :, n:] = math.nan
            x[b, :, n::2] = math.inf
    q0, k0, v0, do0 = (x.nan_to_num(0, 0, 0) for x in (q, k, v, dout))
    mask = dict(sinks=sinks, window=window, scale=0.125, lengths=lengths)
    out, lse = streaming.sink_attention_forward(q, k, v, **mask)
    grads = streaming.sink_attention_backward(q, k, v, out, dout, lse, **mask)
    want, bounds = window_reference(q0, k0, v0, do0, lengths, window, sinks, 0.125)
    for name, got in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *grads)):
        close(got, want[name], bounds[name], name)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [128, 64, 40])
def test_strides(D):
    """Token-major views with gaps give the bits that packed tensors give; outputs may be views too; gradients accumulate."""
    q, k, v, dout = tensors(2, 6, 2, 190, D, seed=3, token_major=True)
    mask = dict(sinks=3, window=50, scale=0.1)
    first = check_window(q, k, v, dout, None, 50, 3, 0.1)
    room = torch.full((2, 190, 9, D), 7.0, device=DEVICE)
    out, lse = streaming.sink_attention_forward(q.contiguous(), k.contiguous(), v.contiguous(), **mask, out=room[:, :, 2:8].transpose(1, 2))
    assert torch.equal(out, first[0]) and torch.equal(lse, first[1])
    assert bool((room[:, :, :2] == 7).all()) and bool((room[:, :, 8:] == 7).all())
    start = [torch.randn(x.shape, device=DEVICE) for x in (q, k, v)]
    given = [x.clone() for x in start]
    got = streaming.sink_attention_backward(q, k, v, out, dout, lse, **mask, dq=given[0], dk=given[1], dv=given[2])
    for g, s, fresh in zip(got, start, first[2:]):
        assert torch.equal(g, s + fresh)


@pytest.mark.gpu
def test_broadcast_inputs():
    """Keys and values shared by the sequences of a batch through a stride of 0: the gradients are those of the expanded tensors."""
    q, k, v, dout = tensors(3, 4, 2, 140, 64, seed=14)
    k, v = k[:1].expand(3, -1, -1, -1), v[:1].expand(3, -1, -1, -1)
    check_window(q, k, v, dout, None, 30, 2, 0.125)
    with pytest.raises(GonanoError):
        out, lse = streaming.sink_attention_forward(q, k, v, 2, 30)
        streaming.sink_attention_backward(q, k, v, out, dout, lse, 2, 30, dq=torch.zeros_like(q), dk=torch.zeros(1, 2, 140, 64, device=DEVICE).expand(3, -1, -1, -1),
                                          dv=torch.zeros(3, 2, 140, 64, device=DEVICE))


@pytest.mark.gpu
def test_windows_and_sinks_beyond_every_length():
    big = 2 ** 31 - 1
    q, k, v, dout = tensors(1, 4, 2, 200, 64, seed=15)
    for window, sinks in ((big, 0), (5, big), (big, big)):
        check_window(q, k, v, dout, None, window, sinks, 0.125)
    for counts in ([1, 1], [40, 7]):
        check_paged(counts, [90, 8], 4, 2, 64, 16, big, big)
    cache = Cache(1, 1, 64, 16, 2)   # tokens that stand before the cache, with the widest window
    cache.fill([20])
    x = torch.randn(30, 2, 64, device=DEVICE)
    starts, lens = torch.tensor([0, 30], dtype=torch.int32, device=DEVICE), torch.tensor([20], dtype=torch.int32, device=DEVICE)
    got = [streaming.paged_attention(x, cache.k, cache.v, cache.table, starts, lens, 30, scale=0.125, window=w) for w in (-1, big)]
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


@pytest.mark.gpu
def test_misaligned_views():
    """Tensors that start 4 bytes behind a 16-byte boundary."""
    def shift(x):
        return torch.cat([x.new_zeros(1), x.flatten()])[1:].view(x.shape)
    plain = tensors(1, 4, 2, 140, 64, seed=4)
    a = check_window(*plain, None, 30, 2, 0.2)
    b = check_window(*(shift(x) for x in plain), None, 30, 2, 0.2)
    for x, y in zip(a, b):
        assert torch.equal(x, y)


@pytest.mark.gpu
def test_extreme_magnitudes():
    """Large and small tensors, and keys and values of very different sizes in one sequence."""
    q, k, v, dout = tensors(1, 4, 2, 200, 64, seed=5)
    check_window(q * 1e8, k * 1e-8, v * 1e20, dout * 1e-15, None, 64, 4, 0.125)
    check_window(q * 1e-12, k * 1e12, v * 1e-20, dout * 1e10, None, 64, 4, 0.125)
    steps = torch.logspace(-6, 0, 200, device=DEVICE)[:, None]
    check_window(q, k * steps, v * steps.flip(0), dout, None, -1, 0, 0.125)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [16, 64, 128])
@pytest.mark.parametrize("B", [37, 77, 113])
def test_many_short_sequences_with_slow_stores(B, D):
    """Two to six pieces of one key tile for every SM, whose queries are at hand long before the last results are stored (a word at a time)."""
    H, Hkv, T = 8, 2, 106
    q, k, v, _ = tensors(B, H, Hkv, T, D)
    store = torch.empty(B, H, T, D + 1, device=DEVICE)
    got = [torch.zeros(1, device=DEVICE)]
    for window, sinks in [(0, 0), (20, 1)]:
        out, lse = streaming.sink_attention_forward(q, k, v, sinks, window, 0.25, out=store[..., :D])
        at = torch.arange(T, device=DEVICE)
        see = visible(at, at, window, sinks)
        for b in (0, B // 2, B - 1):
            for h in range(Hkv):
                mine = slice(h * 4, h * 4 + 4)
                qq, kk, vv = (x.double() for x in (q[b, mine], k[b, h], v[b, h]))
                want, wlse, w = attend64(qq, kk, vv, see, 0.25)
                e = 2 * score_bound(qq, kk, 0.25)
                close(out[b, mine], want, (e + PRODUCT) * torch.einsum("gnm,md->gnd", w, vv.abs()) + FLOOR * (see.double() @ vv.abs() + 2 * float(vv.abs().max())), "out")
                close(lse[b, mine], wlse, (e + PRODUCT) * (1 + wlse.abs()), "lse")
        first = out.clone()
        for _ in range(50):
            streaming.sink_attention_forward(q, k, v, sinks, window, 0.25, out=store[..., :D])
            got.append((out != first).sum())
    assert int(torch.stack([x.reshape(()).float() for x in got]).sum()) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("which", ["k", "v"])
def test_non_finite_key_reaches_only_its_queries(value, which):
    q, k, v, _ = tensors(1, 2, 1, 400, 64, seed=6)
    clean, clean_lse = streaming.sink_attention_forward(q, k, v, sinks=2, window=20, scale=0.125)
    (k if which == "k" else v)[0, 0, 150, 3] = value
    out, lse = streaming.sink_attention_forward(q, k, v, sinks=2, window=20, scale=0.125)
    hit = torch.zeros(400, dtype=torch.bool, device=DEVICE)
    hit[150:171] = True
    # an infinite key's score may be -inf, a weight of 0 by the formula; every other case shows in channel 3 of all that see the key
    if which == "v" or math.isnan(value):
        assert not bool(out[0, :, hit, 3].isfinite().any())
    close(out[0, :, ~hit], clean[0, :, ~hit].double(), 2.0 ** -16, "out")
    close(lse[0, :, ~hit], clean_lse[0, :, ~hit].double(), 2.0 ** -16, "lse")


@pytest.mark.gpu
def test_gradient_against_differences():
    """Directional derivative of sum(out * dout) by central differences of the forward."""
    q, k, v, dout = tensors(1, 4, 2, 90, 32, seed=7)
    mask = dict(sinks=3, window=20, scale=0.2)
    out, lse = streaming.sink_attention_forward(q, k, v, **mask)
    grads = streaming.sink_attention_backward(q, k, v, out, dout, lse, **mask)
    gen = torch.Generator(device=DEVICE).manual_seed(8)
    steps = [torch.randn(x.shape, generator=gen, device=DEVICE) for x in (q, k, v)]
    h = 2.0 ** -7
    ends = [streaming.sink_attention_forward(*(x + s * h * d for x, d in zip((q, k, v), steps)), **mask)[0].double() for s in (1, -1)]
    numeric = float(((ends[0] - ends[1]) * dout.double()).sum() / (2 * h))
    analytic = float(sum((g.double() * d.double()).sum() for g, d in zip(grads, steps)))
    # third-order term of the differences: h^2 / 6 times a third derivative of the size of the sum's terms; float32 forward / h
    size = float(dout.double().norm() * out.double().norm())
    assert abs(numeric - analytic) <= size * (h * h + 2.0 ** -17 / h)


@pytest.mark.gpu
def test_same_bits_every_time():
    q, k, v, dout = tensors(2, 8, 1, 600, 128, seed=9)
    mask = dict(sinks=4, window=128, scale=0.09)
    runs = []
    for _ in range(3):
        out, lse = streaming.sink_attention_forward(q, k, v, **mask)
        runs.append((out, lse, *streaming.sink_attention_backward(q, k, v, out, dout, lse, **mask)))
    for x, y, z in zip(*runs):
        assert torch.equal(x, y) and torch.equal(x, z)


@pytest.mark.gpu
def test_matches_the_windowed_attention():
    """Without sinks the operator is the framework's windowed attention."""
    from gonano_b200.backend import CudaBackend
    q, k, v, dout = tensors(1, 4, 2, 150, 64, seed=10)
    out, lse = streaming.sink_attention_forward(q, k, v, sinks=0, window=33, scale=1.0)
    o2, l2 = CudaBackend().attention_windowed_forward(*(x.cpu().numpy() for x in (q, k, v)), 0, 33)
    e = 4 * score_bound(q, k, 1.0) + 4 * PRODUCT
    close(out.cpu(), torch.from_numpy(o2).double(), e * float(v.abs().max()), "out")
    close(lse.cpu(), torch.from_numpy(l2).double(), e * (1 + torch.from_numpy(l2).double().abs()), "lse")


# ---------------------------------------------------------------- paged cache

class Cache:
    """Pages, tables and the float64 truth of what every row holds; unused slots are NaN."""

    def __init__(self, rows, kv_heads, dim, page, width, seed=0):
        self.gen = torch.Generator(device=DEVICE).manual_seed(seed)
        pages = rows * width + 2
        self.k = torch.full((pages, kv_heads, page, dim), math.nan, device=DEVICE)
        self.v = torch.full_like(self.k, math.inf)
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))[:rows * width].to(torch.int32)
        self.table = order.view(rows, width).to(DEVICE)
        self.page, self.kv_heads, self.dim, self.rows = page, kv_heads, dim, rows

    def fill(self, lens):
        for r, n in enumerate(lens):
            for j0 in range(0, n, self.page):
                m = min(self.page, n - j0)
                where = int(self.table[r, j0 // self.page])
                self.k[where, :, :m] = torch.randn(self.kv_heads, m, self.dim, generator=self.gen, device=DEVICE)
                self.v[where, :, :m] = torch.randn(self.kv_heads, m, self.dim, generator=self.gen, device=DEVICE)

    def row(self, r, n):
        flat = [p[self.table[r].long()].transpose(1, 2).reshape(-1, self.kv_heads, self.dim)[:n].double() for p in (self.k, self.v)]
        return flat


def check_paged(counts, lens, heads, kv_heads, dim, page, window, sinks, mass=True, append=True, seed=0, scale=None, hide=None, max_query=None):
    rows = len(counts)
    width = max(1, -(-max(lens) // page))
    cache = Cache(rows, kv_heads, dim, page, width, seed)
    cache.fill(lens if not append else [n - c for n, c in zip(lens, counts)])
    scale = 1 / math.sqrt(dim) if scale is None else scale
    used = sum(counts)
    tokens = used + 2
    gen = cache.gen
    q = torch.randn(tokens, heads, dim, generator=gen, device=DEVICE)
    nk, nv = (torch.randn(tokens, kv_heads, dim, generator=gen, device=DEVICE) for _ in range(2))
    starts = torch.tensor([0, *itertools.accumulate(counts)], dtype=torch.int32, device=DEVICE)
    lens_t = torch.tensor(lens, dtype=torch.int32, device=DEVICE)
    table = cache.table.clone()
    if hide is not None:   # (row, table column): a page that does not exist
        table[hide] = -7
    before = torch.rand(rows, kv_heads, width * page, generator=gen, device=DEVICE) if mass else None
    out = torch.full((tokens, heads, dim), 5.0, device=DEVICE)
    lse = torch.full((tokens, heads), 6.0, device=DEVICE)
    kept = before.clone() if mass else None
    got = streaming.paged_attention(q, cache.k, cache.v, table, starts, lens_t, max(counts) if max_query is None else max_query, new_key=nk if append else None,
                                    new_value=nv if append else None, sinks=sinks, window=window, scale=scale, mass=before, mass_out=kept, out=out, lse=lse)
    assert got[0] is out and got[1] is lse
    assert bool((out[used:] == 5).all()) and bool((lse[used:] == 6).all())
    g = heads // kv_heads
    for r in range(rows):
        b, e, n = int(starts[r]), int(starts[r + 1]), lens[r]
        k64, v64 = cache.row(r, n)
        if append and hide is None and e > b:
            assert torch.equal(k64[n - (e - b):], nk[b:e].double()) and torch.equal(v64[n - (e - b):], nv[b:e].double())
        pos = torch.arange(n - (e - b), n, device=DEVICE)
        see = visible(pos, torch.arange(n, device=DEVICE), window, sinks)
        if hide is not None and hide[0] == r:
            gone = torch.arange(n, device=DEVICE) // page == hide[1]
            see = see & ~gone
            k64[gone], v64[gone] = 0.0, 0.0
        for h in range(kv_heads):
            heads_of = slice(h * g, (h + 1) * g)
            qq = q[b:e, heads_of].double().transpose(0, 1)
            o, l, w = attend64(qq, k64[:, h], v64[:, h], see, scale)
            eb = 2 * score_bound(qq, k64[:, h], scale) if qq.numel() else 0.0
            close(out[b:e, heads_of].transpose(0, 1), o, (eb + PRODUCT) * torch.einsum("gnm,md->gnd", w, v64[:, h].abs()) + FLOOR * (n + 2) * float(v64.abs().max() if n else 0), f"out of row {r}")
            close(lse[b:e, heads_of].transpose(0, 1), l, (eb + PRODUCT) * (1 + l.abs()), f"lse of row {r}")
            if mass:
                added = w.sum((0, 1))
                want = added.clone()
                want[:n - (e - b)] += before[r, h, :n - (e - b)].double()
                close(kept[r, h, :n], want, (eb + PRODUCT) * added + 2.0 ** -22 * want.abs(), f"mass of row {r}")
    if mass:
        for r, n in enumerate(lens):
            assert torch.equal(kept[r, :, n:], before[r, :, n:])
    return out, lse, kept


PAGED = [  # counts, lens, heads, kv_heads, dim, page, window, sinks
    ([1], [1], 1, 1, 16, 1, -1, 0),
    ([1], [40], 2, 1, 64, 16, 16, 2),
    ([1] * 9, [1, 2, 15, 16, 17, 33, 64, 100, 384], 6, 2, 128, 16, -1, 0),
    ([1] * 3, [1500, 700, 2049], 8, 1, 128, 64, -1, 0),
    ([1] * 3, [1500, 700, 2049], 8, 1, 128, 24, 600, 5),
    ([1] * 5, [30, 31, 32, 33, 1000], 3, 3, 80, 100, 0, 1),
    ([1, 0, 1, 1], [300, 20, 0, 5], 4, 2, 40, 8, 20, 4),
    ([2, 0, 5, 1], [300, 20, 5, 77], 4, 2, 64, 16, -1, 0),
    ([64, 1, 0, 33, 17], [700, 1, 0, 33, 600], 6, 2, 64, 24, 100, 4),
    ([130, 257], [1000, 257], 8, 1, 128, 64, -1, 0),
    ([200, 3], [999, 1100], 8, 1, 128, 7, 150, 40),
    ([50], [50], 32, 1, 32, 16, -1, 0),
    ([7, 9], [2000, 3], 2, 2, 128, 256, 30, 900),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", [c for c in PAGED if all(n >= m for n, m in zip(c[1], c[0]))])
@pytest.mark.parametrize("mass", [False, True])
def test_paged(case, mass):
    check_paged(*case, mass=mass)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [33, 511, 512])
def test_many_ragged_chunks(rows):
    """Most rows without new tokens, the first and the last ones among them, some with one tile of them and one with several."""
    counts = [0 if r < 2 or r > rows - 3 or r % 7 else r % 5 for r in range(rows)]
    counts[14], counts[rows // 2] = 70, 33
    lens = [max(c, (r * 37) % 90) for r, c in enumerate(counts)]
    check_paged(counts, lens, 8, 2, 32, 16, -1, 0, mass=False)


@pytest.mark.gpu
def test_paged_without_append_and_with_unit_scale():
    check_paged([1, 1], [77, 300], 6, 2, 128, 16, -1, 0, append=False, scale=1.0)
    check_paged([40, 70], [77, 300], 6, 2, 128, 16, -1, 0, append=False, scale=1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("counts", [[1, 1], [90, 33]])
def test_missing_pages_are_not_seen(counts):
    check_paged(counts, [400, 333], 4, 2, 64, 32, -1, 0, append=False, hide=(0, 3))
    check_paged(counts, [400, 333], 4, 2, 64, 32, 60, 5, append=False, hide=(1, 0))


@pytest.mark.gpu
def test_more_tokens_than_keys():
    """The first tokens then stand before the cache: they see nothing."""
    cache = Cache(1, 1, 64, 16, 2)
    cache.fill([20])
    q = torch.randn(30, 2, 64, device=DEVICE)
    starts, lens = torch.tensor([0, 30], dtype=torch.int32, device=DEVICE), torch.tensor([20], dtype=torch.int32, device=DEVICE)
    out, lse = streaming.paged_attention(q, cache.k, cache.v, cache.table, starts, lens, 30, scale=0.125)
    assert bool((out[:10] == 0).all()) and bool((lse[:10] == -math.inf).all()) and bool(out.isfinite().all()) and bool(lse[10:].isfinite().all())


@pytest.mark.gpu
@pytest.mark.parametrize("count", [1, 40])
def test_pages_beyond_32_bits(count):
    """Pages whose elements lie past 2^31 and 2^32: attention, the new tokens' slots and eviction."""
    pages, page, dim, n = 600_000, 64, 128, 300
    k = torch.zeros(pages, 1, page, dim, device=DEVICE)   # 19.7 GB
    v = torch.zeros(pages, 1, page, dim, device=DEVICE)
    gen = torch.Generator(device=DEVICE).manual_seed(16)
    ids = [pages - 1, 270_000, 3, 530_000, pages - 2]
    flat = torch.randn(2, n, dim, generator=gen, device=DEVICE)
    for i, p in enumerate(ids):
        m = min(page, n - count - i * page)
        if m > 0:
            k[p, 0, :m], v[p, 0, :m] = flat[0, i * page:i * page + m], flat[1, i * page:i * page + m]
    table = torch.tensor([ids], dtype=torch.int32, device=DEVICE)
    q = torch.randn(count, 4, dim, generator=gen, device=DEVICE)
    starts, lens = torch.tensor([0, count], dtype=torch.int32, device=DEVICE), torch.tensor([n], dtype=torch.int32, device=DEVICE)
    out, lse, mass = streaming.paged_attention(q, k, v, table, starts, lens, count, new_key=flat[0, n - count:, None], new_value=flat[1, n - count:, None], scale=0.09,
                                               mass_out=torch.zeros(1, 1, 5 * page, device=DEVICE))
    see = visible(torch.arange(n - count, n, device=DEVICE), torch.arange(n, device=DEVICE), -1, 0)
    o, l, w = attend64(q.double().transpose(0, 1), flat[0].double(), flat[1].double(), see, 0.09)
    e = 2 * score_bound(q, flat[0], 0.09) + PRODUCT
    close(out.transpose(0, 1), o, e * torch.einsum("gnm,md->gnd", w, flat[1].double().abs()) + FLOOR * (n + 2) * float(flat[1].abs().max()), "out")
    for i, p in enumerate(ids):
        m = min(page, n - i * page)
        assert torch.equal(k[p, 0, :m], flat[0, i * page:i * page + m]) and torch.equal(v[p, 0, :m], flat[1, i * page:i * page + m])
    fresh = torch.tensor([[pages - 3, 400_000]], dtype=torch.int32, device=DEVICE)
    kept, _, _ = streaming.evict_pages(k, v, mass, table, lens, 100, 4, 10, new_table=fresh)
    got = k[fresh[0].long(), 0].reshape(-1, dim)[:100]
    assert torch.equal(got, flat[0, kept[0, 0].long()])


@pytest.mark.gpu
def test_paged_equals_the_padded_form():
    """A sequence fed in chunks through the cache gives what one pass over it gives."""
    T, heads, kv_heads, dim, page = 300, 8, 2, 64, 16
    q, k, v, _ = tensors(1, heads, kv_heads, T, dim, seed=11)
    mask = dict(sinks=4, window=70, scale=0.125)
    want, want_lse = streaming.sink_attention_forward(q, k, v, **mask)
    cache = Cache(1, kv_heads, dim, page, -(-T // page))
    done = 0
    bound = 4 * (score_bound(q, k, 0.125) + PRODUCT)
    for n in (1, 1, 40, 1, 129, 2, 100, 26):
        part = [x[0, :, done:done + n].transpose(0, 1) for x in (q, k, v)]
        done += n
        out, lse = streaming.paged_attention(part[0], cache.k, cache.v, cache.table, torch.tensor([0, n], dtype=torch.int32, device=DEVICE),
                                             torch.tensor([done], dtype=torch.int32, device=DEVICE), n, new_key=part[1], new_value=part[2], **mask)
        close(out.transpose(0, 1), want[0, :, done - n:done].double(), bound * float(v.abs().max()), f"out at {done}")
        close(lse.transpose(0, 1), want_lse[0, :, done - n:done].double(), bound * (1 + want_lse[0, :, done - n:done].double().abs()), f"lse at {done}")
    assert done == T


# ---------------------------------------------------------------- eviction

def evict64(mass, lens, budget, sinks, recent):
    kept = []
    for r, n in enumerate(lens):
        for h in range(mass.shape[1]):
            values = mass[r, h].tolist()
            if n <= budget:
                kept.append(list(range(n)))
                continue
            key = lambda j: -math.inf if math.isnan(values[j]) else values[j]  # noqa: E731
            order = sorted(range(sinks, n - recent), key=lambda j: (math.isnan(values[j]), -key(j) if not math.isnan(values[j]) else 0.0, j))
            kept.append(sorted([*range(sinks), *order[:budget - sinks - recent], *range(n - recent, n)]))
    return kept


def check_evict(lens, kv_heads, dim, page, budget, sinks, recent, mass_of, in_place, seed=0):
    rows = len(lens)
    width = max(1, -(-max(lens) // page))
    extra = max(1, -(-budget // page))
    cache = Cache(rows, kv_heads, dim, page, width + extra, seed)
    cache.fill(lens)
    table, target = cache.table[:, :width].contiguous(), cache.table[:, width:].contiguous()
    mass = mass_of(torch.rand(rows, kv_heads, width * page, generator=cache.gen, device=DEVICE))
    old = cache.k.clone(), cache.v.clone()
    if in_place and width * page < min(budget, width * page):
        pytest.skip("no room")
    kept, new_lens, moved = streaming.evict_pages(cache.k, cache.v, mass, table, torch.tensor(lens, dtype=torch.int32, device=DEVICE), budget, sinks, recent,
                                                  new_table=None if in_place else target)
    assert new_lens.tolist() == [min(n, budget) for n in lens]
    want = evict64(mass.cpu(), lens, budget, sinks, recent)
    to = table if in_place else target
    touched = torch.zeros(cache.k.shape[:3], dtype=torch.bool, device=DEVICE)
    for r in range(rows):
        for h in range(kv_heads):
            w = want[r * kv_heads + h]
            got = kept[r, h].tolist()
            assert got[:len(w)] == w and all(x == -1 for x in got[len(w):])
            idx = torch.tensor(w, dtype=torch.long, device=DEVICE)
            slots = torch.arange(len(w), device=DEVICE)
            assert torch.equal(moved[r, h, :len(w)].nan_to_num(3.0), mass[r, h, idx].nan_to_num(3.0)) and bool((moved[r, h, len(w):] == 0).all())
            src, dst = table[r].long()[idx // page], to[r].long()[slots // page]
            touched[dst, h, slots % page] = True
            for now, then in zip((cache.k, cache.v), old):
                assert torch.equal(now[dst, h, slots % page], then[src, h, idx % page])
    for now, then in zip((cache.k, cache.v), old):
        assert torch.equal(now[~touched].nan_to_num(9.0), then[~touched].nan_to_num(9.0))


EVICT = [  # lens, kv_heads, dim, page, budget, sinks, recent
    ([384, 300, 128, 100, 0, 1], 2, 64, 16, 128, 1, 33),
    ([2500, 1025], 1, 128, 64, 600, 4, 100),
    ([700, 33], 3, 80, 24, 1, 0, 0),
    ([700, 33], 1, 33, 1, 32, 32, 0),
    ([500, 60], 2, 16, 100, 40, 0, 40),
    ([9, 3], 1, 8, 4, 0, 0, 0),
    ([257, 513], 2, 128, 16, 256, 3, 5),
    ([5000], 1, 4, 256, 4999, 10, 20),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", EVICT)
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("kind", ["spread", "ties", "equal", "odd"])
def test_evict(case, in_place, kind):
    def odd(m):
        m = (m - 0.5) * 1e6
        m[..., ::7], m[..., 1::7], m[..., 2::11], m[..., 3::13], m[..., 4::17] = math.nan, math.inf, -math.inf, -0.0, 0.0
        return m
    kinds = {"spread": lambda m: m, "ties": lambda m: (m * 5).floor(), "equal": lambda m: m * 0 - 2, "odd": odd}
    check_evict(*case, kinds[kind], in_place)


@pytest.mark.gpu
def test_evict_more_keys_than_are_cached():
    check_evict([60000, 49153], 1, 4, 256, 5000, 4, 100, lambda m: (m * 1000).floor(), False)


@pytest.mark.gpu
def test_evict_bad_pages():
    """Pages that do not exist are neither read nor written: a key from one leaves zeros."""
    cache = Cache(1, 1, 32, 8, 8)
    cache.fill([32])
    table, target = cache.table[:, :4].clone(), cache.table[:, 4:].clone()
    table[0, 1], target[0, 1] = 10 ** 6, -1
    mass = torch.zeros(1, 1, 32, device=DEVICE)
    mass[0, 0, 8:20] = 1.0
    lens = torch.tensor([32], dtype=torch.int32, device=DEVICE)
    old = cache.k.clone()
    kept, _, _ = streaming.evict_pages(cache.k, cache.v, mass, table, lens, 12, new_table=target)
    assert kept[0, 0].tolist() == list(range(8, 20))
    assert bool((cache.k[int(target[0, 0]), 0] == 0).all())
    others = [p for p in range(cache.k.shape[0]) if p != int(target[0, 0])]
    assert torch.equal(cache.k[others].nan_to_num(9.0), old[others].nan_to_num(9.0))


# ---------------------------------------------------------------- together, streams, graphs

def rollout(steps, streams=None):
    """A prompt in chunks, decode steps that gather weights, an eviction into fresh pages, more steps; every output."""
    rows, heads, kv_heads, dim, page = 3, 6, 2, 64, 16
    gen = torch.Generator(device=DEVICE).manual_seed(12)
    width, small = 20, 8
    k = torch.full((rows * (width + small), kv_heads, page, dim), math.nan, device=DEVICE)
    v = torch.full_like(k, math.nan)
    ids = torch.randperm(rows * (width + small), generator=torch.Generator().manual_seed(3)).to(torch.int32).view(rows, -1).to(DEVICE)
    table, second = ids[:, :width].contiguous(), ids[:, width:].contiguous()
    mass = torch.zeros(rows, kv_heads, width * page, device=DEVICE)
    truth = [([], []) for _ in range(rows)]
    lens, results = [0] * rows, []

    def step(counts, table, mass, keep):
        for r, c in enumerate(counts):
            lens[r] += c
        tokens = sum(counts)
        q, nk, nv = (torch.randn(tokens, h, dim, generator=gen, device=DEVICE) for h in (heads, kv_heads, kv_heads))
        starts = torch.tensor([0, *itertools.accumulate(counts)], dtype=torch.int32, device=DEVICE)
        out, lse, _ = streaming.paged_attention(q, k, v, table, starts, torch.tensor(lens, dtype=torch.int32, device=DEVICE), max(counts), new_key=nk, new_value=nv,
                                                scale=0.125, mass=mass, mass_out=mass)
        results.append((q, nk, nv, counts, out, lse))

    step([100, 61, 0], table, mass, None)
    step([60, 100, 150], table, mass, None)
    for _ in range(steps):
        step([1, 1, 1], table, mass, None)
    kept, new_lens, moved = streaming.evict_pages(k, v, mass, table, torch.tensor(lens, dtype=torch.int32, device=DEVICE), budget=96, sinks=4, recent=32, new_table=second)
    results.append((kept, mass.clone(), list(lens)))
    lens[:] = new_lens.tolist()
    mass2 = torch.zeros(rows, kv_heads, small * page, device=DEVICE)
    mass2[:, :, :96] = moved
    for _ in range(steps):
        step([1, 1, 1], second, mass2, None)
    return results


@pytest.mark.gpu
def test_rollout_with_eviction():
    rows, heads, kv_heads, dim, g = 3, 6, 2, 64, 3
    results = rollout(5)
    held = [[torch.zeros(0, dim, dtype=torch.float64, device=DEVICE) for _ in range(2 * kv_heads)] for _ in range(rows)]
    mass = [[torch.zeros(0, dtype=torch.float64, device=DEVICE) for _ in range(kv_heads)] for _ in range(rows)]
    for item in results:
        if len(item) == 3:   # the eviction: checked against its own weights, then applied
            kept, weights, lens = item
            want = evict64(weights.cpu(), lens, 96, 4, 32)
            for r, h in itertools.product(range(rows), range(kv_heads)):
                w = want[r * kv_heads + h]
                assert kept[r, h, :len(w)].tolist() == w
                close(weights[r, h, :lens[r]], mass[r][h], 2.0 ** -12 * (1 + mass[r][h]), "mass")   # per step 2 e + 2^-18 with e = 2^-19 * 8.5 * 8.5 / 8... < 2^-15, 7 steps
                for half in range(2):
                    held[r][half * kv_heads + h] = held[r][half * kv_heads + h][w]
                mass[r][h] = mass[r][h][w]
            continue
        q, nk, nv, counts, out, lse = item
        at = 0
        for r, c in enumerate(counts):
            for h in range(kv_heads):
                held[r][h] = torch.cat([held[r][h], nk[at:at + c, h].double()])
                held[r][kv_heads + h] = torch.cat([held[r][kv_heads + h], nv[at:at + c, h].double()])
                n = held[r][h].shape[0]
                pos = torch.arange(n - c, n, device=DEVICE)
                qq = q[at:at + c, h * g:(h + 1) * g].double().transpose(0, 1)
                o, l, w = attend64(qq, held[r][h], held[r][kv_heads + h], visible(pos, torch.arange(n, device=DEVICE), -1, 0), 0.125)
                if c:
                    e = 2 * score_bound(qq, held[r][h], 0.125) + PRODUCT
                    close(out[at:at + c, h * g:(h + 1) * g].transpose(0, 1), o, e * torch.einsum("gnm,md->gnd", w, held[r][kv_heads + h].abs()) + FLOOR * (n + 2) * float(held[r][kv_heads + h].abs().max()), "out")
                    close(lse[at:at + c, h * g:(h + 1) * g].transpose(0, 1), l, e * (1 + l.abs()), "lse")
                mass[r][h] = torch.cat([mass[r][h], torch.zeros(c, dtype=torch.float64, device=DEVICE)]) + w.sum((0, 1))
            at += c


@pytest.mark.gpu
def test_runs_on_the_current_stream():
    """Inputs made on a side stream are used there, without a wait for the device."""
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        q, k, v, dout = tensors(2, 4, 2, 256, 64, seed=13)
        check_window(q, k, v, dout, None, 50, 4, 0.125)
    side.synchronize()


TRAINING = [  # B, H, Hkv, T, D, window, sinks, ragged: planes of a cluster, of two launches, key tiles in parts, tiny ones
    (5, 6, 2, 150, 128, 40, 3, True),
    (1, 8, 1, 2100, 128, 256, 5, False),
    (1, 2, 1, 1500, 64, -1, 0, True),
    (9, 2, 1, 20, 40, 5, 1, True),
]


def training_pass(case, seed):
    B, H, Hkv, T, D, window, sinks, ragged = case
    q, k, v, dout = tensors(B, H, Hkv, T, D, seed=seed)
    lengths = torch.tensor([(T * (b + 1)) // B for b in range(B)], dtype=torch.int32, device=DEVICE) if ragged else None
    mask = dict(sinks=sinks, window=window, scale=0.1, lengths=lengths)

    def run():
        out, lse = streaming.sink_attention_forward(q, k, v, **mask)
        grads = streaming.sink_attention_backward(q, k, v, out, dout, lse, **mask)
        return [x * 1.0 for x in (out, lse, *grads)]   # what a following kernel reads
    return (q, k, v, dout), run


@pytest.mark.gpu
def test_training_passes_behind_one_another():
    """Nothing waits on the host between calls, which take over one another's memory."""
    passes = [training_pass(case, seed)[1] for seed, case in enumerate(TRAINING)]
    alone = []
    for run in passes:
        alone.append(run())
        torch.cuda.synchronize()
    for _ in range(10):
        got = [run() for run in passes]
        for want, have in zip(alone, got):
            for x, y in zip(want, have):
                assert torch.equal(x, y)


@pytest.mark.gpu
@pytest.mark.parametrize("case", TRAINING)
def test_captured_training_pass(case):
    inputs, run = training_pass(case, 3)
    run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        captured = run()
    for step in range(3):
        for x in inputs:
            x.mul_(1.0 + 0.25 * step)
        graph.replay()
        replayed = [x.clone() for x in captured]
        for x, y in zip(replayed, run()):
            assert torch.equal(x, y)


@pytest.mark.gpu
def test_two_graphs_at_once():
    """Two captured calls replayed on two streams at once give what eager calls give, on the inputs that stand there at replay."""
    sets, graphs, outs = [], [], []
    for i in range(2):
        q, k, v, dout = tensors(2, 8, 2, 300 + 100 * i, 128, seed=20 + i)
        mask = dict(sinks=4, window=90, scale=0.09)
        nk = torch.randn(2, 2, 128, device=DEVICE)
        cache = Cache(2, 2, 128, 16, 45, seed=i)
        cache.fill([500, 400 + i])
        table, fresh = cache.table[:, :32].contiguous(), cache.table[:, 32:].contiguous()
        starts = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEVICE)
        lens = torch.tensor([501, 401 + i], dtype=torch.int32, device=DEVICE)
        mass = torch.zeros(2, 2, 512, device=DEVICE)
        q1 = torch.randn(2, 8, 128, device=DEVICE)

        def call(q=q, k=k, v=v, dout=dout, q1=q1, nk=nk, cache=cache, table=table, fresh=fresh, starts=starts, lens=lens, mass=mass, mask=mask):
            out, lse = streaming.sink_attention_forward(q, k, v, **mask)
            grads = streaming.sink_attention_backward(q, k, v, out, dout, lse, **mask)
            paged = streaming.paged_attention(q1, cache.k, cache.v, table, starts, lens, 1, new_key=nk, new_value=nk, scale=0.09, mass=mass, mass_out=torch.zeros_like(mass))
            kept = streaming.evict_pages(cache.k, cache.v, paged[2], table, lens, 200, 4, 20, new_table=fresh)
            return [out, lse, *grads, *paged, *kept]
        call()   # warm-up before the capture
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call())
        graphs.append(graph)
        sets.append((q, k, v, dout, call))
    for q, k, v, dout, _ in sets:
        for x in (q, k, v, dout):
            x.mul_(0.5)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for (_, _, _, _, call), got in zip(sets, outs):
        for x, y in zip(got, call()):
            assert torch.equal(x, y)


# ---------------------------------------------------------------- refusals

def sink_params(**over):
    p = _lib.GnSinkParams(batch=2, n_head=4, n_kv_head=2, seq=8, head_dim=64, sinks=1, window=4, scale=1.0)
    for n, x in over.items():
        setattr(p, n, x)
    return p


def paged_params(**over):
    p = _lib.GnPagedParams(rows=2, tokens=2, max_query=1, max_context=32, n_head=4, n_kv_head=2, head_dim=64, page_size=16, pages=4, table_width=2, window=-1, scale=1.0)
    for n, x in over.items():
        setattr(p, n, x)
    return p


def evict_params(**over):
    p = _lib.GnEvictParams(rows=2, n_kv_head=2, head_dim=64, page_size=16, pages=4, table_width=2, new_width=2, mass_stride=32, max_context=32, budget=16, sinks=1, recent=2)
    for n, x in over.items():
        setattr(p, n, x)
    return p


@pytest.fixture(scope="module")
def lib():
    from gonano_b200 import build
    build.build()
    return _lib.load()


@pytest.mark.parametrize("over", [dict(head_dim=0), dict(head_dim=129), dict(n_kv_head=3), dict(n_kv_head=0), dict(n_head=0), dict(batch=-1), dict(seq=-1), dict(sinks=-1),
                                  dict(scale=math.nan), dict(scale=math.inf), dict(batch=70000), dict(query=_lib.GnView(None, -1, 1, 1)), dict(seq=2 ** 30)])
def test_sink_refusals(lib, over):
    import ctypes as C
    n = C.c_int64()
    view = _lib.GnView(None, 64, 64, 64)
    assert lib.gn_attention_sink_workspace(C.byref(sink_params(**over)), 1, C.byref(n)) == 1
    assert lib.gn_attention_sink_forward(C.byref(sink_params(**over)), C.byref(view), None, None, 0, None) == 1
    assert lib.gn_attention_sink_backward(C.byref(sink_params(**over)), *[C.byref(view)] * 2, None, *[C.byref(view)] * 3, 0, None, 0, None) == 1
    assert b"attention_sink" in lib.gn_last_error()


def test_null_arguments_are_refused(lib):
    import ctypes as C
    n = C.c_int64()
    view = _lib.GnView(None, 64, 64, 64)
    assert lib.gn_attention_sink_workspace(C.byref(sink_params()), 0, None) == 1
    assert lib.gn_attention_sink_workspace(None, 0, C.byref(n)) == 1
    assert lib.gn_attention_sink_forward(C.byref(sink_params()), C.byref(view), None, None, 0, None) == 1
    assert lib.gn_attention_sink_forward(C.byref(sink_params()), None, None, None, 0, None) == 1
    assert lib.gn_attention_sink_backward(C.byref(sink_params()), None, None, None, None, None, None, 0, None, 0, None) == 1
    assert lib.gn_attention_paged(C.byref(paged_params()), C.byref(view), None, None, 0, None) == 1
    assert lib.gn_attention_paged(None, None, None, None, 0, None) == 1
    assert lib.gn_cache_evict(C.byref(evict_params()), None, None, None, None) == 1
    assert lib.gn_cache_evict(None, None, None, None, None) == 1


@pytest.mark.parametrize("over", [dict(head_dim=129), dict(n_kv_head=3), dict(rows=-1), dict(tokens=-1), dict(page_size=0), dict(max_context=33), dict(max_context=-1),
                                  dict(sinks=-2), dict(scale=math.nan), dict(rows=70000), dict(table_width=2 ** 30), dict(max_query=-1)])
def test_paged_refusals(lib, over):
    import ctypes as C
    n = C.c_int64()
    view = _lib.GnView(None, 64, 64, 64)
    assert lib.gn_attention_paged_workspace(C.byref(paged_params(**over)), C.byref(n)) == 1
    assert lib.gn_attention_paged(C.byref(paged_params(**over)), C.byref(view), None, None, 0, None) == 1
    assert b"attention_paged" in lib.gn_last_error()


@pytest.mark.parametrize("over", [dict(budget=2), dict(budget=-1), dict(sinks=-1), dict(recent=-1), dict(max_context=33), dict(mass_stride=31), dict(new_width=0),
                                  dict(page_size=0), dict(rows=-1), dict(rows=40000), dict(sinks=2 ** 31 - 1, recent=2 ** 31 - 1)])
def test_evict_refusals(lib, over):
    import ctypes as C
    assert lib.gn_cache_evict(C.byref(evict_params(**over)), None, None, None, None) == 1
    assert b"cache_evict" in lib.gn_last_error()


def test_empty_calls_need_no_device(lib):
    import ctypes as C
    view = _lib.GnView(None, 64, 64, 64)
    assert lib.gn_attention_sink_forward(C.byref(sink_params(batch=0)), C.byref(view), None, None, 0, None) == 0
    assert lib.gn_attention_sink_backward(C.byref(sink_params(seq=0)), *[C.byref(view)] * 2, None, *[C.byref(view)] * 3, 0, None, 0, None) == 0
    assert lib.gn_attention_paged(C.byref(paged_params(rows=0)), C.byref(view), None, None, 0, None) == 0
    assert lib.gn_cache_evict(C.byref(evict_params(rows=0)), None, None, None, None) == 0


def test_host_tensors_are_refused():
    x = torch.zeros(1, 2, 4, 8)
    with pytest.raises(GonanoError):
        streaming.sink_attention_forward(x, x, x, 0, -1)
    with pytest.raises(GonanoError):
        streaming.paged_attention(x[0], x, x, torch.zeros(1, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), 1)
    with pytest.raises(GonanoError):
        streaming.evict_pages(x, x, x[0], torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), 1)


@pytest.mark.gpu
def test_wrong_tensors_are_refused(lib):
    import ctypes as C
    q, k, v, dout = tensors(1, 4, 2, 16, 32)
    with pytest.raises(GonanoError):
        streaming.sink_attention_forward(q.half(), k, v, 0, -1)
    with pytest.raises(GonanoError):
        streaming.sink_attention_forward(q, k[:, :, :8], v, 0, -1)
    with pytest.raises(GonanoError):
        streaming.sink_attention_forward(q, k.cpu(), v, 0, -1)
    with pytest.raises(GonanoError):
        streaming.sink_attention_forward(q.transpose(2, 3).contiguous().transpose(2, 3), k, v, 0, -1)
    with pytest.raises(GonanoError):
        streaming.sink_attention_forward(q, k, v, 0, -1, out=q[:, :1].expand(1, 4, 16, 32))   # elements of out share memory
    out, lse = streaming.sink_attention_forward(q, k, v, 0, -1)
    with pytest.raises(GonanoError):
        streaming.sink_attention_backward(q, k, v, out, dout, lse, 0, -1, dq=q.clone())
    host = torch.zeros(1, 4, 16, 32)
    p = _lib.GnSinkParams(_lib.GnView(host.data_ptr(), 2048, 512, 32), *[_lib.GnView(x.data_ptr(), 1024, 512, 32) for x in (k, v)], 1, 4, 2, 16, 32, 0, -1, 1.0)
    view = _lib.GnView(out.data_ptr(), 2048, 512, 32)
    assert lib.gn_attention_sink_forward(C.byref(p), C.byref(view), lse.data_ptr(), None, 0, None) == 1
    assert b"not device memory" in lib.gn_last_error()
    p.query = _lib.GnView(q.data_ptr(), 2048, 512, 32)
    views = [C.byref(_lib.GnView(x.data_ptr(), x.shape[1] * 512, 512, 32)) for x in (q.clone(), k.clone(), v.clone())]
    assert lib.gn_attention_sink_backward(C.byref(p), C.byref(view), C.byref(view), lse.data_ptr(), *views, 0, None, 0, None) == 1
    assert b"workspace" in lib.gn_last_error()
