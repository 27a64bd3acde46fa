"""Cases of the streaming-attention operators: attention with a sliding window and a few first keys that stay visible
(training and prefill), attention of new tokens over a paged cache (single tokens and chunks), and eviction from that cache by
accumulated attention weight.

``run`` computes an operator in its plain form, or, where ``own`` is true, by the framework's calls.  Query i sees key j when
j <= i and (window < 0 or i - j <= window or j < sinks), both within the sequence; positions count from the start of the cache.
"""
import math

import torch

own = False

DEVICE = "cuda"


def listed():
    return [
        # a training pass of the dense d12 preset's heads: many short ragged rollouts in one padded batch
        {"name": "train_d12", "kind": "train", "batch": 64, "seq": 383, "heads": 6, "kv_heads": 2, "dim": 128, "window": 128, "sinks": 4, "ragged": True},
        # a long-context training pass with eight query heads on one key head
        {"name": "train_long", "kind": "train", "batch": 2, "seq": 8704, "heads": 8, "kv_heads": 1, "dim": 128, "window": 512, "sinks": 4, "ragged": False},
        # the plumbing model's heads: the smallest training step, where launches count
        {"name": "train_plumbing", "kind": "train", "batch": 8, "seq": 63, "heads": 2, "kv_heads": 1, "dim": 64, "window": 16, "sinks": 1, "ragged": True},
        # a head dimension between the powers of two, an odd length and the whole causal context
        {"name": "train_odd", "kind": "train", "batch": 3, "seq": 2049, "heads": 12, "kv_heads": 4, "dim": 80, "window": -1, "sinks": 0, "ragged": True},
        # the prefill of long prompts
        {"name": "prefill_long", "kind": "prefill", "batch": 4, "seq": 8192, "heads": 8, "kv_heads": 1, "dim": 128, "window": 512, "sinks": 64, "ragged": False},
        # one decode step of the d12 rollout's 512 rows
        {"name": "decode_d12", "kind": "paged", "rows": 512, "chunk": 1, "context": 384, "heads": 6, "kv_heads": 2, "dim": 128, "page": 16, "window": -1, "sinks": 0, "mass": False},
        # one decode step over long caches, keeping the weights that an eviction will rank by
        {"name": "decode_long", "kind": "paged", "rows": 32, "chunk": 1, "context": 8704, "heads": 8, "kv_heads": 1, "dim": 128, "page": 64, "window": -1, "sinks": 0, "mass": True},
        # the smallest call: one row, one token
        {"name": "decode_one", "kind": "paged", "rows": 1, "chunk": 1, "context": 40, "heads": 2, "kv_heads": 1, "dim": 64, "page": 16, "window": 16, "sinks": 2, "mass": False},
        # a chunk of a long prompt over what is cached of it
        {"name": "chunk_long", "kind": "paged", "rows": 4, "chunk": 512, "context": 8704, "heads": 8, "kv_heads": 1, "dim": 128, "page": 64, "window": -1, "sinks": 0, "mass": False},
        # ragged chunks (some of them empty), pages of an odd size, a window with sinks, weights kept
        {"name": "chunk_mixed", "kind": "paged", "rows": 24, "chunk": 64, "context": 2000, "heads": 6, "kv_heads": 2, "dim": 64, "page": 24, "window": 700, "sinks": 4, "mass": True},
        # shrinking long caches to a quarter
        {"name": "evict_long", "kind": "evict", "rows": 32, "context": 8704, "kv_heads": 1, "dim": 128, "page": 64, "budget": 2048, "sinks": 4, "recent": 512},
        # shrinking short caches of the plumbing model's kind
        {"name": "evict_short", "kind": "evict", "rows": 8, "context": 384, "kv_heads": 2, "dim": 64, "page": 16, "budget": 128, "sinks": 1, "recent": 33},
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["train", "train", "prefill", "paged", "paged", "paged", "evict"])
    kv_heads, dim = rng.choice([1, 2, 3, 4]), rng.choice([16, 40, 64, 80, 96, 128, 128, 128])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 8])
    if kind in ("train", "prefill"):
        seq = _spread(rng, 1, 8704)
        most = (2 * 8 * 8704 * 8704) // (4 * heads * max(seq, 64) ** 2)   # a quarter of the longest listed pass
        while most < 1:
            seq, most = seq // 2, most * 4 + 1
        return {"kind": kind, "batch": _spread(rng, 1, max(1, min(96, most))), "seq": seq, "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "window": rng.choice([-1, 0, _spread(rng, 1, 1500)]), "sinks": rng.choice([0, 1, 4, _spread(rng, 1, 300)]), "ragged": rng.random() < 0.5}
    context = _spread(rng, 2, 8704)
    page = rng.choice([1, 8, 16, 24, 64, 100, 256])
    if kind == "paged":
        chunk = rng.choice([1, 1, _spread(rng, 1, 512)])
        chunk = min(chunk, context)
        most = min((32 * 8704) // (kv_heads * context), (4 * 512 * 8 * 8704) // (heads * chunk * context))
        return {"kind": kind, "rows": _spread(rng, 1, max(1, min(512, most))), "chunk": chunk, "context": context, "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "page": page, "window": rng.choice([-1, -1, _spread(rng, 1, 1500)]), "sinks": rng.choice([0, 4, _spread(rng, 1, 100)]), "mass": rng.random() < 0.5}
    budget = _spread(rng, 1, context)
    sinks = min(rng.choice([0, 1, 4, 64]), budget)
    return {"kind": kind, "rows": _spread(rng, 1, max(1, min(64, (32 * 8704) // (kv_heads * context)))), "context": context, "kv_heads": kv_heads, "dim": dim, "page": page,
            "budget": budget, "sinks": sinks, "recent": rng.randint(0, budget - sinks)}


# ---------------------------------------------------------------- what a user's program has in hand

def _ints(generator, low, high, n):
    return torch.randint(low, high + 1, (n,), generator=generator, dtype=torch.int32)


def _unit(x):
    """Rows of root mean square 1.2, as the model's normalised queries and keys are."""
    return x * (1.2 / x.square().mean(-1, keepdim=True).sqrt())


def _normal(generator, *shape):
    return torch.randn(*shape, generator=generator, device=DEVICE, dtype=torch.float32)


def prepare(case, seed):
    host = torch.Generator().manual_seed(seed)
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    state = dict(case)
    dim, kv_heads = case["dim"], case["kv_heads"]
    state["scale"] = 1.0 / math.sqrt(dim)
    if case["kind"] in ("train", "prefill"):
        batch, seq, heads = case["batch"], case["seq"], case["heads"]
        state["q"] = _unit(_normal(gen, batch, heads, seq, dim))
        state["k"] = _unit(_normal(gen, batch, kv_heads, seq, dim))
        state["v"] = _normal(gen, batch, kv_heads, seq, dim)
        state["lengths"] = _ints(host, (seq + 1) // 2, seq, batch).to(DEVICE) if case["ragged"] else None
        if case["kind"] == "train":
            state["dout"] = _normal(gen, batch, heads, seq, dim) * 1e-3
        return state
    rows, page, context = case["rows"], case["page"], case["context"]
    per_row = -(-context // page)
    if case["kind"] == "paged":
        heads, chunk = case["heads"], case["chunk"]
        # ragged chunks whose sum does not go by the seed: the first row's is whole, the second's empty, the others make pairs
        counts = torch.ones(rows, dtype=torch.int32)
        if chunk > 1:
            counts = _ints(host, 0, chunk, rows)
            counts[1::2] = chunk - counts[0:rows - 1:2]
            counts[0], counts[1:2], counts[rows - 1:] = chunk, 0, chunk if rows % 2 else counts[rows - 1]
        lens = torch.maximum(_ints(host, max(1, context // 2), context, rows), counts)
        lens[0] = context
        starts = torch.zeros(rows + 1, dtype=torch.int32)
        starts[1:] = counts.cumsum(0)
        used = int(starts[-1])
        tokens = used + (3 if chunk > 1 else 0)   # a buffer may be longer than what is in it
        pages = rows * per_row + 3
        order = torch.randperm(pages, generator=host)[:rows * per_row].to(torch.int32)
        state.update(pages=pages, tokens=tokens, used=used, table=order.view(rows, per_row).to(DEVICE), starts=starts.to(DEVICE), lens=lens.to(DEVICE),
                     q=_unit(_normal(gen, tokens, heads, dim)), new_key=_unit(_normal(gen, tokens, kv_heads, dim)), new_value=_normal(gen, tokens, kv_heads, dim),
                     out=torch.zeros(tokens, heads, dim, device=DEVICE), lse=torch.zeros(tokens, heads, device=DEVICE))
        if case["mass"]:
            state["weights"] = torch.rand(rows, kv_heads, per_row * page, generator=gen, device=DEVICE) * 4
            state["weights_out"] = torch.zeros_like(state["weights"])
    else:
        kept = -(-case["budget"] // page)
        lens = _ints(host, max(1, context // 2), context, rows)
        lens[0] = context
        pages = rows * (per_row + kept) + 3
        order = torch.randperm(pages, generator=host)[:rows * (per_row + kept)].to(torch.int32).view(rows, per_row + kept)
        # weights as a rollout leaves them: most keys little, a few much; halved steps make some of them equal
        weights = torch.rand(rows, kv_heads, per_row * page, generator=gen, device=DEVICE).pow(8) * 50
        state.update(pages=pages, table=order[:, :per_row].contiguous().to(DEVICE), new_table=order[:, per_row:].contiguous().to(DEVICE), lens=lens.to(DEVICE),
                     weights=(weights * 64).round() / 64)
    state["key_pages"] = _unit(_normal(gen, state["pages"], kv_heads, page, dim))
    state["value_pages"] = _normal(gen, state["pages"], kv_heads, page, dim)
    return state


# ---------------------------------------------------------------- plain forms

def _visible(position, keys, state):
    """Truth values [..., queries, keys] from positions [..., queries] and key indices [keys]."""
    i, j = position[..., :, None], keys
    see = j <= i
    if state["window"] >= 0:
        see = see & ((i - j <= state["window"]) | (j < state["sinks"]))
    return see


def _softmax(scores, see):
    """Weights and log-sum-exp of the visible scores; a row that sees nothing has weights 0 and -inf."""
    scores = scores.masked_fill(~see, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = top.masked_fill(top == -math.inf, 0.0)
    weights = (scores - top).exp()
    total = weights.sum(-1, keepdim=True)
    return weights / total.masked_fill(total == 0, 1.0), (top + total.log()).squeeze(-1)


def _plain_window(state):
    batch, seq, heads, kv_heads, dim = (state[n] for n in ("batch", "seq", "heads", "kv_heads", "dim"))
    group = heads // kv_heads
    at = torch.arange(seq, device=DEVICE)
    see = _visible(at, at, state).expand(batch, seq, seq)
    if state["lengths"] is not None:
        within = at < state["lengths"][:, None]
        see = see & within[:, :, None] & within[:, None, :]
    see = see[:, None, None]
    q = state["q"].view(batch, kv_heads, group, seq, dim)
    k, v = state["k"][:, :, None], state["v"][:, :, None]
    weights, lse = _softmax(torch.matmul(q, k.transpose(-1, -2)) * state["scale"], see)
    out = torch.matmul(weights, v)
    if state["kind"] == "prefill":
        return out.view(batch, heads, seq, dim), lse.view(batch, heads, seq)
    dout = state["dout"].view(batch, kv_heads, group, seq, dim)
    dv = torch.matmul(weights.transpose(-1, -2), dout).sum(2)
    dscores = torch.matmul(dout, v.transpose(-1, -2)) - (dout * out).sum(-1, keepdim=True)
    dscores = dscores * weights * state["scale"]
    dq = torch.matmul(dscores, k)
    dk = torch.matmul(dscores.transpose(-1, -2), q).sum(2)
    return out.view(batch, heads, seq, dim), lse.view(batch, heads, seq), dq.view(batch, heads, seq, dim), dk, dv


def _plain_paged(state):
    rows, chunk, heads, kv_heads, dim, page = (state[n] for n in ("rows", "chunk", "heads", "kv_heads", "dim", "page"))
    group, used = heads // kv_heads, state["used"]
    table, starts, lens = state["table"].long(), state["starts"].long(), state["lens"].long()
    token = torch.arange(used, device=DEVICE)
    row = torch.bucketize(token, starts[1:], right=True)
    position = lens[row] - (starts[row + 1] - token)
    where, slot = table[row, position // page], position % page
    state["key_pages"][where, :, slot] = state["new_key"][:used]
    state["value_pages"][where, :, slot] = state["new_value"][:used]
    keys = table.shape[1] * page
    k = state["key_pages"][table].permute(0, 2, 1, 3, 4).reshape(rows, kv_heads, 1, keys, dim)
    v = state["value_pages"][table].permute(0, 2, 1, 3, 4).reshape(rows, kv_heads, 1, keys, dim)
    offset = token - starts[row]
    q = torch.zeros(rows, chunk, heads, dim, device=DEVICE)
    q[row, offset] = state["q"][:used]
    q = q.view(rows, chunk, kv_heads, group, dim).permute(0, 2, 3, 1, 4)
    step = torch.arange(chunk, device=DEVICE)
    count = starts[1:] - starts[:-1]
    at = lens[:, None] - count[:, None] + step
    see = _visible(at, torch.arange(keys, device=DEVICE), state) & (step < count[:, None])[:, :, None]
    weights, lse = _softmax(torch.matmul(q, k.transpose(-1, -2)) * state["scale"], see[:, None, None])
    out = torch.matmul(weights, v).permute(0, 3, 1, 2, 4).reshape(rows, chunk, heads, dim)[row, offset]
    lse = lse.permute(0, 3, 1, 2).reshape(rows, chunk, heads)[row, offset]
    state["out"][:used], state["lse"][:used] = out, lse
    answer = [state["out"], state["lse"], state["key_pages"], state["value_pages"]]
    if state["mass"]:
        added = weights.sum((2, 3))
        j = torch.arange(keys, device=DEVICE)
        old = (j < (lens - count)[:, None])[:, None]
        live = (j < lens[:, None])[:, None]
        answer.append(torch.where(live, torch.where(old, state["weights"], 0.0) + added, 0.0))
    return answer


def _plain_evict(state):
    rows, kv_heads, page, budget = (state[n] for n in ("rows", "kv_heads", "page", "budget"))
    lens = state["lens"].long()
    keys = state["table"].shape[1] * page
    j = torch.arange(keys, device=DEVICE)
    forced = (j < state["sinks"]) | (j >= (lens - state["recent"])[:, None])
    rank = state["weights"].masked_fill(forced[:, None], math.inf).masked_fill((j >= lens[:, None])[:, None], -math.inf)
    first = rank.sort(dim=-1, descending=True, stable=True).indices[..., :budget]
    new_lens = lens.clamp(max=budget)
    slots = torch.arange(first.shape[-1], device=DEVICE)
    live = (slots < new_lens[:, None])[:, None].expand_as(first)
    kept = torch.where(live, first, keys).sort(-1).values
    kept = torch.where(live, kept, -1)
    source, row = kept.clamp(min=0), torch.arange(rows, device=DEVICE)[:, None, None]
    head = torch.arange(kv_heads, device=DEVICE)[None, :, None]
    moved = torch.where(live, state["weights"].gather(-1, source), 0.0)
    from_page = state["table"].long()[row, source // page]
    to_page = state["new_table"].long()[row, slots // page].expand_as(kept)
    to_slot, heads = (slots % page).expand_as(kept), head.expand_as(kept)
    for pages in (state["key_pages"], state["value_pages"]):
        old = pages[to_page, heads, to_slot]
        pages[to_page, heads, to_slot] = torch.where(live[..., None], pages[from_page, heads, source % page], old)
    pad = budget - kept.shape[-1]
    kept = torch.nn.functional.pad(kept, (0, pad), value=-1)
    return [kept.int(), new_lens.int(), torch.nn.functional.pad(moved, (0, pad)), state["key_pages"], state["value_pages"]]


# ---------------------------------------------------------------- one pass

def run(state):
    if own:
        from gonano_b200 import streaming
        if state["kind"] in ("train", "prefill"):
            mask = dict(sinks=state["sinks"], window=state["window"], scale=state["scale"], lengths=state["lengths"])
            out, lse = streaming.sink_attention_forward(state["q"], state["k"], state["v"], **mask)
            if state["kind"] == "prefill":
                return out, lse
            return (out, lse, *streaming.sink_attention_backward(state["q"], state["k"], state["v"], out, state["dout"], lse, **mask))
        if state["kind"] == "paged":
            answer = streaming.paged_attention(
                state["q"], state["key_pages"], state["value_pages"], state["table"], state["starts"], state["lens"], max_query=state["chunk"],
                max_context=state["context"], new_key=state["new_key"], new_value=state["new_value"], sinks=state["sinks"], window=state["window"],
                scale=state["scale"], mass=state.get("weights"), mass_out=state.get("weights_out"), out=state["out"], lse=state["lse"])
            return [*answer[:2], state["key_pages"], state["value_pages"], *answer[2:]]
        kept, lens, mass = streaming.evict_pages(state["key_pages"], state["value_pages"], state["weights"], state["table"], state["lens"], budget=state["budget"],
                                                 sinks=state["sinks"], recent=state["recent"], new_table=state["new_table"], max_context=state["context"])
        return [kept, lens, mass, state["key_pages"], state["value_pages"]]
    if state["kind"] in ("train", "prefill"):
        return _plain_window(state)
    return _plain_paged(state) if state["kind"] == "paged" else _plain_evict(state)


# ---------------------------------------------------------------- what a pass cannot do without

def _pairs(first, last, window, sinks):
    """Visible (query, key) pairs of the queries at positions first .. last - 1."""
    total = 0
    if window < 0:
        return (last - first) * (first + last + 1) // 2
    inner = min(last, window + 1 + sinks)   # up to here every earlier key is visible
    if first < inner:
        total += (inner - first) * (first + inner + 1) // 2
    return total + max(0, last - max(first, inner)) * (window + 1 + sinks)


def work(case):
    dim, kv_heads = case["dim"], case["kv_heads"]
    if case["kind"] in ("train", "prefill"):
        batch, seq, heads = case["batch"], case["seq"], case["heads"]
        seq = seq if not case["ragged"] else (3 * seq + 1) // 4   # the mean length
        pairs = batch * heads * _pairs(0, seq, case["window"], case["sinks"])
        tokens = batch * seq
        read = 4 * tokens * dim * (2 * heads + 2 * kv_heads) + 4 * tokens * heads
        if case["kind"] == "prefill":
            return {"bytes": read, "flops": 4 * dim * pairs}
        return {"bytes": read + 4 * tokens * dim * (2 * heads + 2 * kv_heads), "flops": 14 * dim * pairs}
    rows, context = case["rows"], case["context"]
    mean = context if rows == 1 else (context + (rows - 1) * (3 * context // 4)) // rows
    if case["kind"] == "paged":
        heads = case["heads"]
        chunk = case["chunk"] if case["chunk"] == 1 or rows == 1 else max(1, case["chunk"] // 2)   # the mean
        seen = mean if case["window"] < 0 else min(mean, case["window"] + case["sinks"] + chunk)
        pairs = rows * heads * _pairs(max(0, mean - chunk), mean, case["window"], case["sinks"])
        size = rows * (8 * dim * kv_heads * seen + 8 * chunk * dim * (heads + 2 * kv_heads) + 4 * chunk * heads)
        return {"bytes": size + (8 * rows * kv_heads * seen if case["mass"] else 0), "flops": 4 * dim * pairs}
    kept = min(case["budget"], mean)
    return {"bytes": rows * kv_heads * (4 * mean + kept * (16 * dim + 8)), "flops": 0}


# ---------------------------------------------------------------- the definition, in 64 bits

def _exact_row(q, k, v, positions, window, sinks, scale):
    """One (sequence, key head): q [group, queries, dim], k / v [keys, dim], in float64: output, weights, log-sum-exp."""
    keys = torch.arange(k.shape[0], device=q.device)
    hidden = keys[None, :] > positions[:, None]
    if window >= 0:
        hidden |= (positions[:, None] - keys[None, :] > window) & (keys[None, :] >= sinks)
    scores = torch.einsum("gqd,kd->gqk", q, k) * scale
    scores = scores.masked_fill(hidden, -math.inf)
    lse = torch.logsumexp(scores, -1)
    weights = torch.softmax(scores, -1)
    return torch.einsum("gqk,kd->gqd", weights, v), weights, lse


def exact(case, seed):
    state = prepare(case, seed)
    dim, kv_heads, scale = case["dim"], case["kv_heads"], state["scale"]
    if case["kind"] in ("train", "prefill"):
        group = case["heads"] // kv_heads
        q, k, v = (state[n].double() for n in ("q", "k", "v"))
        out = torch.zeros_like(q)
        lse = torch.full(q.shape[:3], -math.inf, dtype=torch.float64, device=DEVICE)
        grads = [torch.zeros_like(x) for x in (q, k, v)]
        for b in range(case["batch"]):
            n = case["seq"] if state["lengths"] is None else int(state["lengths"][b])
            for h in range(kv_heads):
                mine = slice(h * group, (h + 1) * group)
                leaves = [x.clone().requires_grad_(case["kind"] == "train") for x in (q[b, mine, :n], k[b, h, :n], v[b, h, :n])]
                o, _, l = _exact_row(*leaves, torch.arange(n, device=DEVICE), case["window"], case["sinks"], scale)
                out[b, mine, :n], lse[b, mine, :n] = o.detach(), l.detach()
                if case["kind"] == "train":
                    got = torch.autograd.grad(o, leaves, state["dout"][b, mine, :n].double())
                    grads[0][b, mine, :n], grads[1][b, h, :n], grads[2][b, h, :n] = got
        return (out, lse) if case["kind"] == "prefill" else (out, lse, *grads)
    page = case["page"]
    table, lens = state["table"].tolist(), state["lens"].tolist()
    pages = [state["key_pages"].double(), state["value_pages"].double()]
    if case["kind"] == "paged":
        starts, group = state["starts"].tolist(), case["heads"] // kv_heads
        out = torch.zeros(state["tokens"], case["heads"], dim, dtype=torch.float64, device=DEVICE)
        lse = torch.zeros(state["tokens"], case["heads"], dtype=torch.float64, device=DEVICE)
        mass = torch.zeros(case["rows"], kv_heads, len(table[0]) * page, dtype=torch.float64, device=DEVICE) if case["mass"] else None
        for r in range(case["rows"]):
            begin, end, n = starts[r], starts[r + 1], lens[r]
            mine = torch.tensor(table[r], device=DEVICE)
            flat = []
            for store, new in zip(pages, (state["new_key"], state["new_value"])):
                seq = store[mine].transpose(1, 2).reshape(-1, kv_heads, dim)
                seq[n - (end - begin):n] = new[begin:end].double()
                store[mine] = seq.view(len(table[r]), page, kv_heads, dim).transpose(1, 2)
                flat.append(seq[:n])
            positions = torch.arange(n - (end - begin), n, device=DEVICE)
            for h in range(kv_heads):
                heads = slice(h * group, (h + 1) * group)
                o, w, l = _exact_row(state["q"][begin:end, heads].double().transpose(0, 1), flat[0][:, h], flat[1][:, h], positions, case["window"], case["sinks"], scale)
                out[begin:end, heads], lse[begin:end, heads] = o.transpose(0, 1), l.transpose(0, 1)
                if mass is not None:
                    mass[r, h, :n] = w.sum((0, 1))
                    mass[r, h, :n - (end - begin)] += state["weights"][r, h, :n - (end - begin)].double()
        return [out, lse, *pages] + ([mass] if mass is not None else [])
    new_table, budget = state["new_table"].tolist(), case["budget"]
    kept = torch.full((case["rows"], kv_heads, budget), -1, dtype=torch.int32)
    mass = torch.zeros(case["rows"], kv_heads, budget, dtype=torch.float64)
    weights = state["weights"].double().cpu()
    for r in range(case["rows"]):
        n = lens[r]
        for h in range(kv_heads):
            if n <= budget:
                keep = list(range(n))
            else:
                middle = range(case["sinks"], n - case["recent"])
                values = weights[r, h].tolist()
                heavy = sorted(middle, key=lambda x: (-values[x], x))[:budget - case["sinks"] - case["recent"]]
                keep = sorted([*range(case["sinks"]), *heavy, *range(n - case["recent"], n)])
            keep = torch.tensor(keep)
            kept[r, h, :len(keep)] = keep.int()
            mass[r, h, :len(keep)] = weights[r, h, keep]
            slot = torch.arange(len(keep))
            source, target = torch.tensor(table[r])[keep // page], torch.tensor(new_table[r])[slot // page]
            for store in pages:
                store[target.to(DEVICE), h, (slot % page).to(DEVICE)] = store[source.to(DEVICE), h, (keep % page).to(DEVICE)]
    return [kept.to(DEVICE), torch.tensor([min(n, budget) for n in lens], dtype=torch.int32, device=DEVICE), mass.to(DEVICE), *pages]
