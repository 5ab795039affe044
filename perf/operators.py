"""Cases of the linear recurrence and of the page cache: their inputs, their plain forms and what they cannot do without.

`run` computes an operator in its plain form with elementary torch operations, or, where `own` is
true, with the calls that a user makes of thrust_amd.  `exact` gives the same outputs from the
definitions, in 64 bits and one step (one row, one page) at a time.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
DEVICE = "cuda"


# ---------------------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------------------
def listed():
    return [
        # one short prompt through one narrow layer: latency
        dict(name="scan_short_f32", op="scan", batch=1, rows=33, channels=512, type="f32", gate="f32", log=False, packed=0),
        # one very long document through one layer, gates and inputs in 16 bits and side by side as one projection leaves them
        dict(name="scan_long_bf16", op="scan", batch=1, rows=131072, channels=2048, type="bf16", gate="bf16", log=False, packed=0, fused=True),
        # a training step of one layer: logarithms of the gates in 32 bits, activations in 16
        dict(name="grad_dense_bf16", op="grad", batch=8, rows=4096, channels=2560, type="bf16", gate="f32", log=True, packed=0),
        # a training step on packed sequences of very different lengths (empty ones among them), an odd width
        dict(name="grad_packed_f16", op="grad", batch=1, rows=12345, channels=1111, type="f16", gate="f16", log=False, packed=61),
        # one token for each of a few sequences
        dict(name="step_small_bf16", op="step", batch=8, channels=1024, slots=64, type="bf16", gate="f32", log=True),
        # one token for each sequence of a large batch
        dict(name="step_large_bf16", op="step", batch=2048, channels=8192, slots=4096, type="bf16", gate="bf16", log=False),
        # beams over recurrent states: one page a sequence, always partly filled, so each fork is a copy
        dict(name="fork_states", op="fork", pools=8, pages=512, page=2048, page_size=1 << 20, sequences=256, max_pages=1, pairs=48, share=True),
        # parallel samples of long prompts: full pages are shared, the last one is copied in every layer's keys and values
        dict(name="fork_pages", op="fork", pools=48, pages=4096, page=8192, page_size=16, sequences=1024, max_pages=128, pairs=500, share=True),
        # a scheduler's step on a small server: a few sequences end, others come in their places, not all of which find room
        dict(name="resize_small", op="resize", pools=2, pages=300, page=256, page_size=16, sequences=64, max_pages=40, pairs=9, fill=1.0),
        # the same on a large one
        dict(name="resize_large", op="resize", pools=2, pages=1 << 20, page=16, page_size=16, sequences=4096, max_pages=512, pairs=1500, fill=0.4),
        # a fragmented cache of states is closed up
        dict(name="compact_states", op="compact", pools=4, pages=777, page=1030, page_size=1 << 20, sequences=700, max_pages=1, live=0.4),
        # a fragmented cache of keys and values, a third of it in use, is closed up
        dict(name="compact_pages", op="compact", pools=40, pages=4096, page=8192, page_size=16, sequences=512, max_pages=160, live=0.35),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return min(high, max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["scan", "grad", "step", "fork", "resize", "compact"])
    if op in ("scan", "grad"):
        type_ = rng.choice(["f32", "f16", "bf16"])
        rows, channels = _spread(rng, 1, 60000), _spread(rng, 1, 6000)
        packed = rng.choice([0, 0, _spread(rng, 1, 200)])
        most = 1 << (26 if op == "scan" else 25)
        rows = max(1, min(rows, most // channels))
        batch = 1 if packed else min(_spread(rng, 1, 64), max(1, most // (rows * channels)))
        gate = rng.choice([type_, "f32"])
        return dict(op=op, batch=batch, rows=rows, channels=channels, type=type_, gate=gate, log=rng.random() < 0.5, packed=packed, fused=gate == type_ and rng.random() < 0.5)
    if op == "step":
        type_ = rng.choice(["f32", "f16", "bf16"])
        batch, channels = _spread(rng, 1, 2000), _spread(rng, 1, 8000)
        return dict(op=op, batch=batch, channels=channels, slots=batch + _spread(rng, 1, 1000), type=type_, gate=rng.choice([type_, "f32"]), log=rng.random() < 0.5)
    states = rng.random() < 0.3
    pools, page = rng.randint(1, 40), _spread(rng, 1, 4000)
    pages = _spread(rng, 300, max(301, min(100000, (1 << 28) // (pools * page))))
    case = dict(op=op, pools=pools, pages=pages, page=page, page_size=(1 << 20) if states else rng.choice([1, 7, 16, 64]),
                sequences=min(pages, _spread(rng, 40, 2000)), max_pages=1 if states else _spread(rng, 2, 200))
    if op == "fork":
        return dict(case, pairs=_spread(rng, 1, max(1, case["sequences"] // 3)), share=rng.random() < 0.7)
    if op == "resize":
        return dict(case, pairs=_spread(rng, 1, case["sequences"]), fill=rng.choice([0.4, 0.8, 1.5]))
    return dict(case, live=rng.uniform(0.05, 0.95))


# ---------------------------------------------------------------------------------------
# The inputs
# ---------------------------------------------------------------------------------------
def _gates(shape, kind, log, g):
    """Gates as a trained recurrence has them: most remember tens to thousands of steps, some forget at once."""
    keep = torch.empty(shape, device=DEVICE).uniform_(-7.0, 0.5, generator=g).exp_().neg_()  # log of the gate
    return (keep if log else keep.exp_()).to(TYPES[kind])


def _kind(case):
    """States are kept in 32 bits, keys and values in 16."""
    return torch.float32 if case["page_size"] == 1 << 20 else torch.bfloat16


def _tables(case, seed, g):
    """Lengths, tables and counts of a cache in use: sequence s holds its pages in tables[s], an even one shares its first pages with the odd one before it."""
    sequences, most, size, pages = case["sequences"], case["max_pages"], case["page_size"], case["pages"]
    r = torch.Generator().manual_seed(seed)
    op, pairs = case["op"], case.get("pairs", 0)
    budget = pages * (case["live"] if op == "compact" else 0.45)
    mean = max(1.0, min(float(most), budget / sequences))
    held = (torch.rand(sequences, generator=r) * 2 * mean).long().clamp(0, most)  # pages of a sequence
    if most == 1:
        held = (torch.rand(sequences, generator=r) < min(1.0, budget / sequences)).long()
    order = torch.randperm(sequences, generator=r)
    if op == "fork":  # children first: empty; parents behind them: not
        held[order[:pairs]] = 0
        held[order[pairs:]] = held[order[pairs:]].clamp(min=1)
    ends = held.cumsum(0)
    held = torch.where(ends <= int(pages * (0.5 if op != "compact" else max(0.05, case["live"]))), held, 0)
    starts = held.cumsum(0) - held
    ids = torch.randperm(pages, generator=r).int()
    column = torch.arange(most)[None]
    tables = torch.where(column < held[:, None], ids[(starts[:, None] + column).clamp(max=pages - 1)], -1)
    lengths = ((held - 1).clamp(min=0) * size + 1 + (torch.rand(sequences, generator=r) * (size - 1)).long()) * (held > 0)
    if op != "fork":  # prompts in common: the full pages of an odd sequence stand in front of the even one's own
        odd, even = tables[1::2], tables[0::2][: tables[1::2].shape[0]]
        shared = torch.minimum(lengths[1::2] // size, (held[0::2][: odd.shape[0]] - 1).clamp(min=0)) // 2
        even.copy_(torch.where(column < shared[:, None], odd, even))
    refs = torch.zeros(pages + 1, dtype=torch.int32).index_put_((torch.where(tables < 0, pages, tables).long().flatten(),), torch.ones(1, dtype=torch.int32), accumulate=True)[:pages]
    return tables.int().to(DEVICE), lengths.int().to(DEVICE), refs.to(DEVICE), order, held


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    op = case["op"]
    state = {"case": case}
    if op in ("scan", "grad", "step"):
        type_, rows = TYPES[case["type"]], case.get("rows", 1)
        wide = (case["batch"], rows, case["channels"])
        if op == "step" or case["packed"]:
            wide = (case["batch"] * rows, case["channels"])
        state["x"] = torch.randn(wide, device=DEVICE, generator=g).to(type_)
        state["gate"] = _gates(wide, case["gate"], case["log"], g)
        if case.get("fused"):  # the two halves of one projection
            state["gate"], state["x"] = torch.cat([state["gate"], state["x"]], -1).chunk(2, -1)
        if op == "step":
            state["pool"] = torch.randn((case["slots"], case["channels"]), device=DEVICE, generator=g)
            state["slots"] = torch.randperm(case["slots"], device=DEVICE, generator=g)[: case["batch"]].int()
            return state
        state["offsets"] = None
        sequences = case["batch"]
        if case["packed"]:
            sequences = case["packed"]
            r = torch.Generator().manual_seed(seed)
            cuts = (torch.rand(sequences - 1, generator=r) ** 2 * (rows + 1)).long().sort().values
            cuts[1::7] = cuts[0::7][: cuts[1::7].numel()]  # empty sequences
            state["offsets"] = torch.cat([torch.zeros(1).long(), cuts.sort().values, torch.tensor([rows])]).int().to(DEVICE)
        state["init"] = torch.randn((sequences, case["channels"]), device=DEVICE, generator=g)
        if op == "grad":
            state["grad_out"] = torch.randn(wide, device=DEVICE, generator=g).to(type_)
            state["grad_final"] = torch.randn((sequences, case["channels"]), device=DEVICE, generator=g)
        return state
    tables, lengths, refs, order, held = _tables(case, seed, g)
    kind = _kind(case)
    pools = [torch.randn((case["pages"], case["page"]), device=DEVICE, generator=g).to(kind) for _ in range(case["pools"])]
    n = case.get("pairs", 0)
    state.update(tables=tables, lengths=lengths, refs=refs, pools=pools)
    if op == "fork":
        parents = order[n:]
        r = torch.Generator().manual_seed(seed + 1)
        state["children"] = order[:n].int().to(DEVICE)
        state["parents"] = parents[torch.randint(0, len(parents), (n,), generator=r)].int().to(DEVICE)
    if op == "resize":
        r = torch.Generator().manual_seed(seed + 1)
        most = case["max_pages"] * case["page_size"]
        mean = min(most, max(1, int(case["pages"] * case["fill"] / n * case["page_size"])))
        state["sequences"] = order[:n].int().to(DEVICE)
        state["lengths_new"] = (torch.rand(n, generator=r) * 2 * mean).long().clamp(1, most).int().to(DEVICE)
    if op == "compact":
        state["tables_new"], state["refs_new"] = torch.empty_like(tables), torch.empty_like(refs)
    if own:
        import thrust_amd

        state["cache"] = thrust_amd.PageCache(pools, case["page_size"], case["sequences"], case["max_pages"], tables=tables, lengths=lengths, refs=refs)
    return state


# ---------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------
def _affine(a, x):
    """Composes the maps h -> a h + x along dim 0 in place by doubling: afterwards (a, x)[t] is the composition of the maps 0 .. t."""
    step = 1
    while step < a.shape[0]:
        x[step:] = torch.addcmul(x[step:], a[step:], x[:-step])
        a[step:] = a[step:] * a[:-step]
        step *= 2
    return a, x


def _rows_of(state):
    """Rows first: [rows, sequences, channels], or [rows, 1, channels] packed, with the heads (first rows of a sequence) of the latter."""
    if state["offsets"] is None:
        return lambda v: v.transpose(0, 1), lambda v: v.transpose(0, 1)
    return lambda v: v.unsqueeze(1), lambda v: v.squeeze(1)


def _plain_scan(state):
    first, back = _rows_of(state)
    a = state["gate"].float()
    a = first(a.exp() if state["case"]["log"] else a).contiguous().clone()
    x = first(state["x"].float()).contiguous().clone()
    gate, init, offsets = a.clone(), state["init"], state["offsets"]
    if offsets is None:
        x[0] += a[0] * init
        before = init
    else:
        begin, end = offsets[:-1].long(), offsets[1:].long()
        some = (end > begin).nonzero().flatten()
        head = begin[some]
        x[head, 0] += a[head, 0] * init[some]
        a[head] = 0.0
        before = init[some]
    h = _affine(a, x)[1]
    shifted = torch.roll(h, 1, 0)
    if offsets is None:
        shifted[0] = before
        final = h[-1].clone()
    else:
        shifted[head, 0] = before
        final = init.clone()
        final[some] = h[end[some] - 1, 0]
    return back(h).to(state["x"].dtype).contiguous(), final, gate, shifted


def _plain_grad(state):
    first, back = _rows_of(state)
    out, final, gate, before = _plain_scan(state)
    init, offsets = state["init"], state["offsets"]
    g = first(state["grad_out"].float()).contiguous().clone()
    a = torch.roll(gate, -1, 0)  # what row t + 1 passes back to row t
    if offsets is None:
        a[-1] = 1.0
        g[-1] += state["grad_final"]
    else:
        begin, end = offsets[:-1].long(), offsets[1:].long()
        some = (end > begin).nonzero().flatten()
        a[end[some] - 1] = 0.0
        g[end[some] - 1, 0] += state["grad_final"][some]
    g = _affine(a.flip(0), g.flip(0))[1].flip(0)
    grad_gate = g * before
    if state["case"]["log"]:
        grad_gate = grad_gate * gate
    if offsets is None:
        grad_init = g[0] * gate[0]
    else:
        grad_init = state["grad_final"].clone()
        grad_init[some] = g[begin[some], 0] * gate[begin[some], 0]
    return {"out": out, "final": final, "grad_gate": back(grad_gate).to(state["gate"].dtype).contiguous(),
            "grad_x": back(g).to(state["x"].dtype).contiguous(), "grad_init": grad_init}


def _plain_step(state):
    a = state["gate"].float()
    a = a.exp() if state["case"]["log"] else a
    slots = state["slots"].long()
    h = a * state["pool"][slots] + state["x"].float()
    state["pool"][slots] = h
    return h.to(state["x"].dtype)


def _plain_free(state, sequences):
    """The sequences give their pages back."""
    tables, refs = state["tables"], state["refs"]
    rows = tables[sequences]
    refs.index_add_(0, rows.clamp(min=0).flatten().long(), -(rows >= 0).int().flatten())
    tables[sequences] = -1
    state["lengths"][sequences] = 0


def _plain_take(state, need):
    """need[i, j]: page j of request i is wanted.  The lowest free pages, in this order; what a request cannot have whole it does not get."""
    wanted = need.sum(1).cumsum(0)
    free = (state["refs"] == 0).nonzero().flatten().int()
    done = (wanted <= free.numel()) | (need.sum(1) == 0)
    rank = need.flatten().cumsum(0).reshape(need.shape) - 1
    taken = need & done[:, None]
    pages = torch.where(taken, free[rank.clamp(0, max(0, free.numel() - 1))] if free.numel() else rank.int(), -1)
    return done, taken, pages


def _plain_fork(state):
    size, most = state["case"]["page_size"], state["case"]["max_pages"]
    children, parents = state["children"].long(), state["parents"].long()
    _plain_free(state, children)
    tables, lengths, refs = state["tables"], state["lengths"], state["refs"]
    column = torch.arange(most, device=DEVICE)[None]
    long = lengths[parents][:, None]
    rows = tables[parents]
    need = (column * size < long) & ((column + 1) * size > long)
    if not state["case"]["share"]:
        need = column * size < long
    done, taken, pages = _plain_take(state, need)
    new = torch.where(done[:, None], torch.where(taken, pages, rows), -1)
    tables[children] = new
    lengths[children] = torch.where(done, long[:, 0], 0)
    refs.index_add_(0, new.clamp(min=0).flatten().long(), (new >= 0).int().flatten())
    source, target = rows[taken].long(), pages[taken].long()
    for pool in state["pools"]:
        pool[target] = pool[source]
    return {"done": done, "tables": tables, "lengths": lengths, "refs": refs, "pools": state["pools"]}


def _plain_resize(state):
    """The sequences that end give their pages back, and what comes in their places gets the lowest free ones."""
    size, most = state["case"]["page_size"], state["case"]["max_pages"]
    sequences, long = state["sequences"].long(), state["lengths_new"]
    _plain_free(state, sequences)
    tables, lengths, refs = state["tables"], state["lengths"], state["refs"]
    need = torch.arange(most, device=DEVICE)[None] * size < long[:, None]
    done, taken, pages = _plain_take(state, need)
    tables[sequences] = pages
    lengths[sequences] = torch.where(done, long, 0)
    refs.index_add_(0, pages.clamp(min=0).flatten().long(), taken.int().flatten())
    return {"done": done, "tables": tables, "lengths": lengths, "refs": refs}


def _plain_compact(state):
    """The highest page in use moves to the lowest free one, and so on, until the pages in use are the lowest ones."""
    tables, refs = state["tables"], state["refs"]
    used = refs > 0
    live = used.sum()
    place = torch.arange(refs.numel(), device=DEVICE)
    target = (~used & (place < live)).nonzero().flatten()
    source = (used & (place >= live)).nonzero().flatten().flip(0)
    for pool in state["pools"]:
        pool[target] = pool[source]
    name = place.int()
    name[source] = target.int()
    state["tables_new"].copy_(torch.where(tables >= 0, name[tables.clamp(min=0).long()], -1))
    state["refs_new"].copy_(torch.where(place < live, refs, 0))
    state["refs_new"][target] = refs[source]
    return {"live": live.int().reshape(1), "tables": state["tables_new"], "refs": state["refs_new"], "pools": state["pools"]}


def _own(state):
    import thrust_amd

    case, op = state["case"], state["case"]["op"]
    if op == "scan":
        out, final = thrust_amd.linear_scan(state["gate"], state["x"], init=state["init"], offsets=state["offsets"], log_gate=case["log"])
        return {"out": out, "final": final}
    if op == "grad":
        out, final, states = thrust_amd.linear_scan(state["gate"], state["x"], init=state["init"], offsets=state["offsets"], log_gate=case["log"], return_states=True)
        grad_gate, grad_x, grad_init = thrust_amd.linear_scan_backward(
            state["grad_out"], state["gate"], state["x"], states, init=state["init"], grad_final=state["grad_final"], offsets=state["offsets"], log_gate=case["log"])
        return {"out": out, "final": final, "grad_gate": grad_gate, "grad_x": grad_x, "grad_init": grad_init}
    if op == "step":
        out = thrust_amd.linear_scan_step(state["gate"], state["x"], state["pool"], slots=state["slots"], log_gate=case["log"])
        return {"out": out, "pool": state["pool"]}
    cache = state["cache"]
    if op == "fork":
        cache.free(state["children"])
        done = cache.fork(state["parents"], state["children"], share=case["share"])
        return {"done": done, "tables": cache.tables, "lengths": cache.lengths, "refs": cache.refs, "pools": state["pools"]}
    if op == "resize":
        cache.free(state["sequences"])
        done = cache.resize(state["sequences"], state["lengths_new"])
        return {"done": done, "tables": cache.tables, "lengths": cache.lengths, "refs": cache.refs}
    live = cache.compact(tables=state["tables_new"], refs=state["refs_new"])
    return {"live": live, "tables": state["tables_new"], "refs": state["refs_new"], "pools": state["pools"]}


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "scan":
        out, final = _plain_scan(state)[:2]
        return {"out": out, "final": final}
    if op == "grad":
        return _plain_grad(state)
    if op == "step":
        return {"out": _plain_step(state), "pool": state["pool"]}
    return _plain_fork(state) if op == "fork" else _plain_resize(state) if op == "resize" else _plain_compact(state)


# ---------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op in ("scan", "grad", "step"):
        e, f = TYPES[case["type"]].itemsize, TYPES[case["gate"]].itemsize
        n = case["batch"] * case.get("rows", 1) * case["channels"]
        if op == "step":
            return {"bytes": n * (f + 2 * e + 8) + 4 * case["batch"], "flops": 2 * n}
        ends = 8 * (case["packed"] or case["batch"]) * case["channels"]
        if op == "scan":
            return {"bytes": n * (f + 2 * e) + ends, "flops": 2 * n}
        return {"bytes": n * (2 * f + 4 * e) + 2 * ends, "flops": 5 * n}
    page, most, n = _kind(case).itemsize * case["page"] * case["pools"], case["max_pages"], case.get("pairs", 0)
    mean = max(1, min(most, int(case["pages"] * 0.45 / case["sequences"])))
    if op == "fork":  # rows of parents and children, the counts searched for free pages, the pages copied
        copied = n * (1 if case["share"] else mean)
        return {"bytes": 2 * copied * page + 8 * n * mean + 4 * case["pages"], "flops": 0}
    if op == "resize":  # rows given back and rows handed out, the counts searched
        return {"bytes": 4 * case["pages"] + 16 * n * mean, "flops": 0}
    live = int(case["live"] * case["pages"])  # pages in use spread evenly: those above the line move
    moved = live * (case["pages"] - live) // case["pages"]
    return {"bytes": 2 * moved * page + 8 * case["pages"] + 8 * case["sequences"] * most, "flops": 0}


# ---------------------------------------------------------------------------------------
# The same outputs from the definitions
# ---------------------------------------------------------------------------------------
def _exact_scan(state):
    """One row after the other in 64 bits."""
    case, offsets = state["case"], state["offsets"]
    a, x = state["gate"].double(), state["x"].double()
    if case["log"]:
        a = a.exp()
    a, x = (v.reshape(-1, case["rows"], case["channels"]) for v in (a, x))
    init = state["init"].double()
    out, before, final = torch.zeros_like(x), torch.zeros_like(x), init.clone()
    spans = [(slice(None), slice(None), 0, case["rows"])]
    if offsets is not None:
        at = offsets.tolist()
        spans = [(0, s, at[s], at[s + 1]) for s in range(len(at) - 1)]
    for b, s, begin, end in spans:
        h = init[s]
        for t in range(begin, end):
            before[b, t] = h
            h = torch.addcmul(x[b, t], a[b, t], h)
            out[b, t] = h
        final[s] = h
    return a, before, out, final, spans


def _exact_grad(state, a, before, spans):
    case = state["case"]
    d = state["grad_out"].double().reshape(a.shape)
    grad_x, grad_init = torch.zeros_like(a), state["grad_final"].double().clone()
    for b, s, begin, end in spans:
        back = state["grad_final"].double()[s]
        for t in range(end - 1, begin - 1, -1):
            g = d[b, t] + back
            grad_x[b, t] = g
            back = a[b, t] * g
        grad_init[s] = back
    grad_gate = grad_x * before * (a if case["log"] else 1.0)
    return grad_gate, grad_x, grad_init


def _exact_pages(state):
    """Page after page, with the tables as lists."""
    case, op, size = state["case"], state["case"]["op"], state["case"]["page_size"]
    tables = [[p for p in row if p >= 0] for row in state["tables"].tolist()]
    lengths, refs = state["lengths"].tolist(), state["refs"].tolist()
    source, target, answer = [], [], {}
    if op == "compact":
        live = sum(r > 0 for r in refs)
        holes = [p for p in range(live) if refs[p] == 0]
        high = [p for p in range(case["pages"] - 1, live - 1, -1) if refs[p] > 0]
        source, target = high, holes
        name = dict(zip(source, target))
        tables = [[name.get(p, p) for p in row] for row in tables]
        for p, q in name.items():
            refs[q], refs[p] = refs[p], 0
        answer["live"] = torch.tensor([live], dtype=torch.int32)
    else:
        named = state["children" if op == "fork" else "sequences"].tolist()
        for s in named:
            for p in tables[s]:
                refs[p] -= 1
            tables[s], lengths[s] = [], 0
        free = [p for p in range(case["pages"]) if refs[p] == 0]
        at, done = 0, []
        wants = state["parents" if op == "fork" else "lengths_new"].tolist()
        for s, w in zip(named, wants):
            long = lengths[w] if op == "fork" else w
            row = list(tables[w]) if op == "fork" else [None] * (-(-long // size))
            wanted = [j for j in range(len(row)) if row[j] is None or not case["share"] or (j + 1) * size > long]
            fits = not wanted or at + len(wanted) <= len(free)
            if fits:
                for k, j in enumerate(wanted):
                    if row[j] is not None:
                        source.append(row[j])
                        target.append(free[at + k])
                    row[j] = free[at + k]
                for p in row:
                    refs[p] += 1
                tables[s], lengths[s] = row, long
            at += len(wanted)
            done.append(fits)
        answer["done"] = torch.tensor(done, dtype=torch.bool)
        answer["lengths"] = torch.tensor(lengths, dtype=torch.int32)
    answer["tables"] = torch.tensor([row + [-1] * (case["max_pages"] - len(row)) for row in tables], dtype=torch.int32)
    answer["refs"] = torch.tensor(refs, dtype=torch.int32)
    if op != "resize":
        moved = [pool.clone() for pool in state["pools"]]
        for new, old in zip(moved, state["pools"]):
            new[target] = old[source]
        answer["pools"] = [p.double() for p in moved]
    return answer


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "step":
        a = state["gate"].double()
        a = a.exp() if case["log"] else a
        pool, slots = state["pool"].double(), state["slots"].tolist()
        out = torch.stack([a[i] * pool[s] + state["x"][i].double() for i, s in enumerate(slots)])
        pool[slots] = out
        return {"out": out, "pool": pool}
    if case["op"] in ("fork", "resize", "compact"):
        return _exact_pages(state)
    a, before, out, final, spans = _exact_scan(state)
    wide = state["x"].shape
    answer = {"out": out.reshape(wide), "final": final}
    if case["op"] == "grad":
        grad_gate, grad_x, grad_init = _exact_grad(state, a, before, spans)
        answer.update(grad_gate=grad_gate.reshape(wide), grad_x=grad_x.reshape(wide), grad_init=grad_init)
    return answer
