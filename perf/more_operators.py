"""Steps of drafted tokens over caches in pages, and the upkeep of such caches, as measured calls.

Each case is one call (or the few that belong together) as a serving program issues it, on inputs
that are already on the GPU.  ``run`` computes it in elementary torch operations in 32 bits, or,
where ``own`` is true, through the library.  Head shapes are this repository's (head_dim 128, 256,
512; GQA 2 to 8; one K = V buffer at head_dim 512), with its 1024-token window.

A cache in pages: a pool [planes, pages, kv heads, page rows, head_dim] (a plane is the K or the V
of a layer), a table [slots, most pages] of the page that holds each run of rows of a sequence (-1:
none), the references to each page, and each sequence's length.

Operators
  tree     a step of 1 .. 64 drafted tokens a sequence, a chain or a tree, over pages
  commit   the accepted tokens' rows moved behind the committed ones in every plane
  fork     sequences made from the first rows of others, and pages for their next rows
  compact  the pages in use moved to the pool's front
  write    rows of a prompt into pages
  read     rows out of pages
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
BF = torch.bfloat16
WINDOW = 1024
EPS = 1e-6


def listed() -> list[dict]:
    return [
        # one user's next token on a sliding layer: the smallest call, latency only
        {"name": "token_b1_local", "op": "tree", "batch": 1, "nodes": 1, "hq": 16, "hkv": 8, "dim": 256, "rows": 1000,
         "page": 16, "window": WINDOW, "chain": True},
        # the next token of a serving batch of ragged lengths
        {"name": "token_b32", "op": "tree", "batch": 32, "nodes": 1, "hq": 32, "hkv": 8, "dim": 128, "rows": 8192,
         "page": 16, "window": 0, "chain": True},
        # a few tokens drafted one behind another for each of eight users
        {"name": "chain5_b8", "op": "tree", "batch": 8, "nodes": 5, "hq": 32, "hkv": 16, "dim": 256, "rows": 8191,
         "page": 64, "window": 0, "chain": True},
        # wide trees of drafted tokens over a K = V layer: the largest call
        {"name": "tree63_b2", "op": "tree", "batch": 2, "nodes": 63, "hq": 32, "hkv": 4, "dim": 512, "rows": 16384,
         "page": 128, "window": 0, "chain": False},
        # a user's accepted path on the layers of a small model
        {"name": "accept_b1", "op": "commit", "batch": 1, "hkv": 4, "dim": 512, "planes": 8, "page": 64, "rows": 1001,
         "accept": 5, "nodes": 24},
        # a serving batch's accepted paths on 24 layers of separate K and V
        {"name": "accept_b32", "op": "commit", "batch": 32, "hkv": 8, "dim": 128, "planes": 48, "page": 16, "rows": 45,
         "accept": 7, "nodes": 33},
        # four beams continue the best one
        {"name": "fork_beams", "op": "fork", "sources": 1, "children": 4, "hkv": 4, "dim": 512, "planes": 8, "page": 64,
         "rows": 2001},
        # eight samples of each of four prompts
        {"name": "fork_samples", "op": "fork", "sources": 4, "children": 32, "hkv": 8, "dim": 128, "planes": 16,
         "page": 32, "rows": 2500},
        # a small pool after a few sequences have ended
        {"name": "compact_small", "op": "compact", "slots": 4, "hkv": 8, "dim": 128, "planes": 4, "page": 16, "rows": 500,
         "spread": 0.4},
        # a serving pool before its front is handed to another model
        {"name": "compact_pool", "op": "compact", "slots": 16, "hkv": 8, "dim": 128, "planes": 16, "page": 64, "rows": 900,
         "spread": 0.5},
        # a prompt's rows of one layer, K and V, behind a shared first part
        {"name": "write_prompt", "op": "write", "batch": 1, "hkv": 16, "dim": 256, "planes": 2, "page": 32, "rows": 4095,
         "past": 777},
        # the rows of a long context, for a chunk's attention over them
        {"name": "read_context", "op": "read", "batch": 1, "hkv": 4, "dim": 512, "planes": 1, "page": 16, "rows": 32767,
         "past": 0},
    ]


def _log_uniform(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng) -> dict:
    op = rng.choice(["tree", "tree", "tree", "tree", "commit", "fork", "compact", "write", "read"])
    dim = rng.choice([128, 256, 512])
    hq, hkv = {128: rng.choice([(32, 8), (16, 8)]), 256: rng.choice([(32, 16), (16, 8)]),
               512: rng.choice([(32, 4), (16, 2)])}[dim]
    page = rng.choice([16, 32, 64, 128])
    if op == "tree":
        nodes = rng.choice([1, _log_uniform(rng, 2, 8), _log_uniform(rng, 2, 64)])
        batch = _log_uniform(rng, 1, 32 if nodes < 9 else 8)
        window = rng.choice([0, 0, WINDOW])
        rows = _log_uniform(rng, 16, 2 * WINDOW if window else 65536 // max(4, batch) if nodes < 9 else 26000 // max(2, batch))
        return {"op": op, "batch": batch, "nodes": nodes, "hq": hq, "hkv": hkv, "dim": dim, "rows": rows, "page": page,
                "window": window, "chain": nodes == 1 or rng.random() < 0.3}
    # planes such that a page of all of them stays within 2 MiB
    planes = min(_log_uniform(rng, 1, 48), max(1, (2 << 20) // (2 * hkv * page * dim)))
    if op == "commit":
        nodes = _log_uniform(rng, 4, 64)
        return {"op": op, "batch": _log_uniform(rng, 1, 32), "hkv": hkv, "dim": dim, "planes": planes, "page": page,
                "rows": _log_uniform(rng, 1, 200), "accept": _log_uniform(rng, 1, min(8, nodes // 2)), "nodes": nodes}
    if op == "fork":
        sources = _log_uniform(rng, 1, 4)
        return {"op": op, "sources": sources, "children": sources * _log_uniform(rng, 1, 8), "hkv": hkv, "dim": dim,
                "planes": planes, "page": page, "rows": _log_uniform(rng, 1, 60 * page)}
    if op == "compact":
        return {"op": op, "slots": _log_uniform(rng, 1, 16), "hkv": hkv, "dim": dim, "planes": planes, "page": page,
                "rows": _log_uniform(rng, 1, 14 * page), "spread": rng.uniform(0.4, 0.9)}
    batch = _log_uniform(rng, 1, 8)
    return {"op": op, "batch": batch, "hkv": hkv, "dim": dim, "planes": rng.choice([1, 2]), "page": page,
            "rows": _log_uniform(rng, 1, 4096 // batch * (512 // dim)), "past": rng.choice([0, _log_uniform(rng, 1, 1000)])}


# ------------------------------------------------------------------------------ inputs

def _gen(seed: int) -> torch.Generator:
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _rms_rows(shape, g, gain: float = 1.0) -> torch.Tensor:
    """bf16 rows of root mean square `gain`: what a q, k or v norm leaves."""
    x = torch.randn(shape, device=DEV, dtype=torch.float32, generator=g)
    x *= gain * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    return x.to(BF)


def _pool(planes: int, pages: int, hkv: int, page: int, dim: int, g) -> torch.Tensor:
    """Random rows, a plane at a time."""
    pool = torch.empty((planes, pages, hkv, page, dim), dtype=BF, device=DEV)
    for plane in pool:
        plane.copy_(_rms_rows(plane.shape, g))
    return pool


def _lengths(batch: int, low: int, high: int, g) -> torch.Tensor:
    """Ragged lengths low .. high, the first one the longest."""
    n = torch.randint(low, high + 1, (batch,), device=DEV, generator=g, dtype=torch.int32)
    n[0] = high
    return n


def _table(rows: torch.Tensor, page: int, most: int, spare: int, g, spread: float = 1.0):
    """(table [slots, most], references [pages]) of sequences of `rows` rows, each on pages of its own, at
    random in a pool of which about `spread` is in use and `spare` pages more."""
    held = (rows.long() + page - 1) // page
    # (sized by the most that the slots can hold, so that a seed does not change the pool)
    pages = int(math.ceil(rows.numel() * most / spread)) + spare
    k = torch.arange(most, device=DEV)
    ids = torch.randperm(pages, device=DEV, generator=g)[:rows.numel() * most].view(-1, most)
    table = torch.where(k < held[:, None], ids, -1).to(torch.int32)
    refs = torch.zeros(pages, dtype=torch.int32, device=DEV)
    refs.index_add_(0, table.clamp(min=0).flatten().long(), (table >= 0).flatten().int())
    return table, refs


def _tree_inputs(case: dict, g) -> dict:
    B, T, hq, hkv, d, R = (case[x] for x in ("batch", "nodes", "hq", "hkv", "dim", "page"))
    length = _lengths(B, max(1, case["rows"] // 8), case["rows"], g)
    most = (case["rows"] + T + R - 1) // R
    table, refs = _table(length + T, R, most, 3, g)
    s = {"q": _rms_rows((B, T, hq, d), g, 2.5), "k_new": _rms_rows((B, T, hkv, d), g), "length": length, "table": table,
         "pool": _pool(1 if d == 512 else 2, refs.numel(), hkv, R, d, g), "parent": None}
    if d != 512:
        s["v_new"] = _rms_rows((B, T, hkv, d), g)
    if not case["chain"]:
        # a node hangs on one of the eight before it; some sequences have fewer nodes
        node = torch.arange(T, device=DEV)
        up = torch.randint(1, 9, (B, T), device=DEV, generator=g)
        parent = torch.where(node == 0, -1, (node - up).clamp(min=0))
        count = torch.randint(max(1, 3 * T // 4), T + 1, (B, 1), device=DEV, generator=g)
        s["parent"] = torch.where(node < count, parent, -2).to(torch.int32)
    return s


def _commit_inputs(case: dict, g) -> dict:
    B, T, A, R = (case[x] for x in ("batch", "nodes", "accept", "page"))
    length = _lengths(B, max(1, case["rows"] // 8), case["rows"], g)
    table, refs = _table(length + T, R, (case["rows"] + T + R - 1) // R, 1, g)
    # paths of a tree whose nodes stand level by level: the first node, then nodes past the first A
    rest = torch.rand((B, T - A), device=DEV, generator=g).argsort(1)[:, :A - 1].sort(1).values + A
    accept = torch.cat([torch.zeros((B, 1), dtype=torch.long, device=DEV), rest], dim=1).to(torch.int32).contiguous()
    count = torch.randint(0, A + 1, (B,), device=DEV, generator=g, dtype=torch.int32)
    count[0] = A
    return {"pool": _pool(case["planes"], refs.numel(), case["hkv"], R, case["dim"], g), "table": table, "refs": refs,
            "start": length, "length": length.clone(), "accept": accept, "count": count}


def _fork_inputs(case: dict, g) -> dict:
    S, n, R = case["sources"], case["children"], case["page"]
    rows = _lengths(S, max(1, case["rows"] // 2), case["rows"], g)
    most = case["rows"] // R + 3
    table, refs = _table(rows, R, most, 3 * n + 2, g)
    table = torch.cat([table, torch.full((n, most), -1, dtype=torch.int32, device=DEV)])
    src = torch.randint(0, S, (n,), device=DEV, generator=g, dtype=torch.int32)
    return {"pool": _pool(case["planes"], refs.numel(), case["hkv"], R, case["dim"], g), "table": table, "refs": refs,
            "length": torch.cat([rows, torch.zeros(n, dtype=torch.int32, device=DEV)]), "src": src,
            "dst": S + torch.arange(n, device=DEV, dtype=torch.int32), "rows": rows[src.long()],
            "next": rows[src.long()] + 1}


def _compact_inputs(case: dict, g) -> dict:
    rows = _lengths(case["slots"], max(1, case["rows"] // 2), case["rows"], g)
    table, refs = _table(rows, case["page"], case["rows"] // case["page"] + 1, 2, g, case["spread"])
    return {"pool": _pool(case["planes"], refs.numel(), case["hkv"], case["page"], case["dim"], g), "table0": table,
            "refs0": refs, "table": table.clone(), "refs": refs.clone(), "length": rows}


def _rows_inputs(case: dict, g) -> dict:
    B, n, R = case["batch"], case["rows"], case["page"]
    row0 = _lengths(B, case["past"] // 2, case["past"], g)
    table, refs = _table(row0 + n, R, (case["past"] + n + R - 1) // R, 1, g)
    s = {"pool": _pool(case["planes"], refs.numel(), case["hkv"], R, case["dim"], g), "table": table, "row0": row0}
    if case["op"] == "write":
        s["rows"] = _rms_rows((case["planes"], B, case["hkv"], n, case["dim"]), g)
    return s


def _inputs(case: dict, seed: int) -> dict:
    make = {"tree": _tree_inputs, "commit": _commit_inputs, "fork": _fork_inputs, "compact": _compact_inputs,
            "write": _rows_inputs, "read": _rows_inputs}[case["op"]]
    return make(case, _gen(seed))


def prepare(case: dict, seed: int) -> dict:
    return {"case": case, **_inputs(case, seed)}


# ------------------------------------------------------------------------------ plain forms

def _place(table: torch.Tensor, rows: torch.Tensor, page: int):
    """(page, row in it) of rows [slots, n] of each slot."""
    at = (rows // page).clamp(0, table.shape[1] - 1)
    return table.gather(1, at).long(), rows % page


def _reach(parent: torch.Tensor) -> torch.Tensor:
    """[B, T, T]: node j is i or above it."""
    T = parent.shape[1]
    up = (parent.unsqueeze(2) == torch.arange(T, device=DEV)).float() + torch.eye(T, device=DEV)
    for _ in range(6):  # paths of up to 64 edges
        up = ((up @ up) > 0).float()
    return up > 0


def _plain_tree(st: dict):
    case = st["case"]
    B, T, hq, hkv, d, R = (case[x] for x in ("batch", "nodes", "hq", "hkv", "dim", "page"))
    G = hq // hkv
    table, length, pool = st["table"], st["length"].long(), st["pool"]
    node = torch.arange(T, device=DEV)
    if st["parent"] is None:
        there = torch.ones((B, T), dtype=torch.bool, device=DEV)
        above = (node <= node.unsqueeze(1)).expand(B, T, T)
    else:
        there = st["parent"] >= -1
        above = _reach(st["parent"]) & there.unsqueeze(2) & there.unsqueeze(1)
    # the new rows behind the committed ones; the row of a node that is none stays
    page, row = _place(table, length.unsqueeze(1) + node, R)
    for plane, new in zip(pool, [st["k_new"]] if d == 512 else [st["k_new"], st["v_new"]]):
        plane[page, :, row] = torch.where(there.view(B, T, 1, 1), new, plane[page, :, row])
    L = table.shape[1] * R

    def held(plane):  # [B, hkv, L, d]
        return plane[table.clamp(min=0).long()].transpose(1, 2).reshape(B, hkv, L, d).float()

    kf = held(pool[0])
    vf = kf if d == 512 else held(pool[1])
    q = st["q"].float().view(B, T, hkv, G, d).permute(0, 2, 3, 1, 4).reshape(B, hkv, G * T, d) * d ** -0.5
    s = (q @ kf.transpose(-1, -2)).view(B, hkv, G, T, L)
    at = torch.arange(L, device=DEV)
    seen = (at < length.view(B, 1, 1)).expand(B, T, L)
    if case["window"]:
        depth = above.sum(2) - 1
        seen = seen & (at > (length.unsqueeze(1) + depth - case["window"]).unsqueeze(2))
    of = at - length.view(B, 1)  # the node in each row
    among = above.gather(2, of.clamp(0, T - 1).unsqueeze(1).expand(B, T, L)) & ((of >= 0) & (of < T)).unsqueeze(1)
    seen = (seen | among) & there.unsqueeze(2)
    s = s.masked_fill(~seen.view(B, 1, 1, T, L), -math.inf)
    top = s.amax(-1, keepdim=True)
    p = (s - torch.where(torch.isinf(top), 0.0, top)).exp()
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    out = (p.view(B, hkv, G * T, L) @ vf).view(B, hkv, G, T, d).permute(0, 3, 1, 2, 4).reshape(B, T, hq, d).to(BF)
    return [out, pool]


def _plain_commit(st: dict):
    R, A = st["case"]["page"], st["case"]["accept"]
    st["length"].copy_(st["start"])  # the step's lengths, as the scheduler hands them over
    length = st["length"].long().unsqueeze(1)
    i = torch.arange(A, device=DEV)
    taken = torch.where(i < st["count"].unsqueeze(1), st["accept"].long(), i)
    page, row = _place(st["table"], length + taken, R)
    rows = st["pool"][:, page, :, row]
    page, row = _place(st["table"], length + i, R)
    st["pool"][:, page, :, row] = rows
    st["length"] += st["count"]
    return [st["pool"], st["length"]]


def _free_pages(refs: torch.Tensor) -> torch.Tensor:
    """The pages nobody holds in order, then the others."""
    return torch.sort((refs != 0).to(torch.int8), stable=True).indices


def _hold(refs: torch.Tensor, pages: torch.Tensor, which: torch.Tensor, by: int) -> None:
    refs.index_add_(0, pages.clamp(min=0).flatten().long(), by * which.flatten().int())


def _plain_fork(st: dict):
    R = st["case"]["page"]
    table, refs, length, pool = st["table"], st["refs"], st["length"], st["pool"]
    src, dst = st["src"].long(), st["dst"].long()
    # what the children held goes back
    old = table[dst]
    _hold(refs, old, old >= 0, -1)
    # full pages are shared
    rows = st["rows"].long()
    full, part = rows // R, rows % R > 0
    k = torch.arange(table.shape[1], device=DEV)
    new = torch.where(k < full.unsqueeze(1), table[src], -1)
    _hold(refs, new, new >= 0, 1)
    # the last rows go to a page of the child's own (a child without: a page onto itself)
    fresh = _free_pages(refs)[(part.long().cumsum(0) - 1).clamp(min=0)]
    last = table[src].gather(1, full.clamp(max=table.shape[1] - 1).unsqueeze(1)).squeeze(1).long()
    last = torch.where(part, last, table[0, 0].long())
    fresh = torch.where(part, fresh, last)
    used = (torch.arange(R, device=DEV) < (rows % R).unsqueeze(1)).view(-1, 1, R, 1)  # the rest of a page stays
    pool[:, fresh] = torch.where(used, pool[:, last], pool[:, fresh])
    _hold(refs, fresh, part, 1)
    new = torch.where((k == full.unsqueeze(1)) & part.unsqueeze(1), fresh.int().unsqueeze(1), new)
    table[dst] = new
    length[dst] = rows.int()
    # pages for the next rows
    to = (st["next"].long() + R - 1) // R
    lack = (k >= full.unsqueeze(1)) & (k < to.unsqueeze(1)) & (new < 0)
    rank = (lack.flatten().long().cumsum(0) - 1).clamp(min=0).view(lack.shape)
    more = _free_pages(refs)[rank]
    table[dst] = torch.where(lack, more.int(), new)
    _hold(refs, more, lack, 1)
    return [pool, table, refs, length]


def _plain_compact(st: dict):
    st["table"].copy_(st["table0"])  # the tables as the scheduler left them
    st["refs"].copy_(st["refs0"])
    table, refs, pool = st["table"], st["refs"], st["pool"]
    at = torch.arange(refs.numel(), device=DEV)
    used = refs > 0
    live = used.sum()
    movers, holes = (used & (at >= live)).nonzero().squeeze(1), (~used & (at < live)).nonzero().squeeze(1)
    pool[:, holes] = pool[:, movers]
    refs[holes] = refs[movers]
    refs[movers] = 0
    at[movers] = holes
    table.copy_(torch.where(table >= 0, at[table.clamp(min=0).long()].int(), -1))
    return [pool, table, refs]


def _plain_rows(st: dict):
    case = st["case"]
    page, row = _place(st["table"], st["row0"].long().unsqueeze(1) + torch.arange(case["rows"], device=DEV), case["page"])
    if case["op"] == "write":
        for plane, rows in zip(st["pool"], st["rows"]):
            plane[page, :, row] = rows.transpose(1, 2)
        return [st["pool"]]
    return [torch.stack([plane[page, :, row].transpose(1, 2) for plane in st["pool"]])]


# ------------------------------------------------------------------------------ the library's calls

def _own_tree(st: dict):
    from apertura_amd.tree import TreeCall, TreeStep

    case, pool = st["case"], st["pool"]
    if "call" not in st:
        step = TreeStep.for_pages(pool[0], st["table"], case["hq"], case["nodes"], window=case["window"],
                                  kv_shared=case["dim"] == 512, scale=case["dim"] ** -0.5)
        st["call"] = TreeCall(step, st["q"], st["k_new"], st.get("v_new"), pool[0], pool[-1], st["length"],
                              table=st["table"], parent=st["parent"])
    return [st["call"](), pool]


def _cache(st: dict):
    from apertura_amd.pages import PagedCache

    if "cache" not in st:
        st["cache"] = PagedCache([st["pool"]], st["table"], st["length"], st.get("refs"))
    return st["cache"]


def _own_commit(st: dict):
    cache = _cache(st)
    st["length"].copy_(st["start"])
    cache.commit(st["accept"], st["count"])
    return [st["pool"], st["length"]]


def _own_fork(st: dict):
    cache = _cache(st)
    cache.fork(st["src"], st["dst"], st["rows"])
    cache.reserve(st["dst"], st["next"])
    return [st["pool"], st["table"], st["refs"], st["length"]]


def _own_compact(st: dict):
    cache = _cache(st)
    st["table"].copy_(st["table0"])
    st["refs"].copy_(st["refs0"])
    cache.compact()
    return [st["pool"], st["table"], st["refs"]]


def _own_rows(st: dict):
    from apertura_amd.pages import pages_read, pages_write

    if st["case"]["op"] == "write":
        pages_write(st["pool"], st["table"], st["row0"], st["rows"])
        return [st["pool"]]
    return [pages_read(st["pool"], st["table"], st["row0"], st["case"]["rows"])]


def run(st: dict):
    op = st["case"]["op"]
    if own:
        return {"tree": _own_tree, "commit": _own_commit, "fork": _own_fork, "compact": _own_compact, "write": _own_rows,
                "read": _own_rows}[op](st)
    return {"tree": _plain_tree, "commit": _plain_commit, "fork": _plain_fork, "compact": _plain_compact,
            "write": _plain_rows, "read": _plain_rows}[op](st)


# ------------------------------------------------------------------------------ work

def work(case: dict) -> dict:
    d, hkv, R = case["dim"], case["hkv"], case["page"]
    row = 2.0 * hkv * d  # bytes of a row of a plane
    if case["op"] == "tree":
        B, T, hq, rows = case["batch"], case["nodes"], case["hq"], case["rows"]
        planes = 1 if d == 512 else 2
        low = max(1, rows // 8)
        lengths = [rows] + [(low + rows) / 2] * (B - 1)  # the mean of what is drawn
        seen = sum(min(n, case["window"] - 1) if case["window"] else n for n in lengths)
        return {"bytes": planes * row * (seen + 2 * B * T) + 4.0 * B * T * hq * d,
                "flops": 4.0 * d * hq * T * (seen + B * T / 4)}
    if case["op"] == "commit":
        moved = case["accept"] - 1 + (case["batch"] - 1) * (case["accept"] - 1) / 2  # the first node's row stays
        return {"bytes": max(16.0 * case["batch"], 2 * case["planes"] * row * moved), "flops": 0.0}
    if case["op"] == "fork":
        n = case["children"]
        pages = case["rows"] // R
        # the last pages' used rows, half a page on average, the tables and the references
        return {"bytes": 2 * case["planes"] * row * n * R / 2 + 8.0 * n * (pages + 2) + 8.0 * case["sources"] * pages,
                "flops": 0.0}
    if case["op"] == "compact":
        most = case["rows"] // R + 1
        held = case["slots"] * most * 0.75
        pool = case["slots"] * most / case["spread"] + 2
        return {"bytes": 2 * case["planes"] * row * R * held * (1 - held / pool) + 8.0 * pool + 8.0 * case["slots"] * most,
                "flops": 0.0}
    return {"bytes": 2 * case["planes"] * row * case["batch"] * case["rows"], "flops": 0.0}


# ------------------------------------------------------------------------------ 64 bits

def _paths(parent: list[int]) -> list[list[int]]:
    """Each node's path from its root, itself last; empty for no node."""
    paths: list[list[int]] = []
    for i, p in enumerate(parent):
        paths.append([i] if p == -1 else paths[p] + [i] if 0 <= p < i and paths[p] else [])
    return paths


def _exact_tree(s: dict, case: dict) -> list:
    T, hq, hkv, d, R = (case[x] for x in ("nodes", "hq", "hkv", "dim", "page"))
    G = hq // hkv
    out = torch.zeros((case["batch"], T, hq, d), dtype=torch.float64, device=DEV)
    for b, n in enumerate(s["length"].tolist()):
        paths = _paths(list(range(-1, T - 1)) if s["parent"] is None else s["parent"][b].tolist())
        pages = s["table"][b, :(n + R - 1) // R].long()
        seen = torch.zeros((T, n + T), dtype=torch.bool, device=DEV)
        for i, path in enumerate(paths):
            if path:
                first = max(0, n + len(path) - case["window"]) if case["window"] else 0
                seen[i, first:n] = True
                seen[i, [n + j for j in path]] = True
        for h in range(hkv):
            k = torch.cat([s["pool"][0][pages, h].reshape(-1, d)[:n], s["k_new"][b, :, h]]).double()
            v = k
            if d != 512:
                v = torch.cat([s["pool"][1][pages, h].reshape(-1, d)[:n], s["v_new"][b, :, h]]).double()
            x = s["q"][b, :, h * G:(h + 1) * G].double() @ k.T / math.sqrt(d)  # [T, G, n + T]
            w = torch.nan_to_num(torch.softmax(torch.where(seen[:, None], x, -math.inf), dim=-1))
            out[b, :, h * G:(h + 1) * G] = w @ v
    return [out, None]


def _exact_commit(s: dict, case: dict) -> list:
    R, pool, length = case["page"], s["pool"].clone(), s["start"].clone()
    for b, (n, c) in enumerate(zip(s["start"].tolist(), s["count"].tolist())):
        pages = s["table"][b].tolist()
        for i, j in enumerate(s["accept"][b, :c].tolist()):
            pool[:, pages[(n + i) // R], :, (n + i) % R] = s["pool"][:, pages[(n + j) // R], :, (n + j) % R]
        length[b] = n + c
    return [pool, length]


def _exact_fork(s: dict, case: dict) -> list:
    R, pool = case["page"], s["pool"].clone()
    table, length = [row[:] for row in s["table"].tolist()], s["length"].tolist()
    refs = s["refs"].tolist()
    lowest = iter([p for p, n in enumerate(refs) if n == 0])  # the children hold nothing
    jobs = list(zip(s["src"].tolist(), s["dst"].tolist(), s["rows"].tolist(), s["next"].tolist()))
    for src, dst, rows, _ in jobs:
        for k in range(rows // R):
            table[dst][k] = table[src][k]
            refs[table[src][k]] += 1
        if rows % R:
            page = next(lowest)
            pool[:, page, :, :rows % R] = s["pool"][:, table[src][rows // R], :, :rows % R]
            table[dst][rows // R], refs[page] = page, 1
        length[dst] = rows
    for _, dst, rows, then in jobs:
        for k in range(rows // R, (then + R - 1) // R):
            if table[dst][k] < 0:
                table[dst][k] = next(lowest)
                refs[table[dst][k]] = 1
    return [pool] + [torch.tensor(x, dtype=torch.int32, device=DEV) for x in (table, refs, length)]


def _exact_compact(s: dict, case: dict) -> list:
    pool, refs = s["pool"].clone(), s["refs0"].tolist()
    live = sum(n > 0 for n in refs)
    to = {}
    for page in range(live, len(refs)):
        if refs[page]:
            to[page] = refs.index(0)
            pool[:, to[page]] = s["pool"][:, page]
            refs[to[page]], refs[page] = refs[page], 0
    table = [[to.get(page, page) for page in row] for row in s["table0"].tolist()]
    return [pool] + [torch.tensor(x, dtype=torch.int32, device=DEV) for x in (table, refs)]


def _exact_rows(s: dict, case: dict) -> list:
    n, R, pool = case["rows"], case["page"], s["pool"].clone()
    rows = s.get("rows")
    if rows is None:
        rows = torch.empty((case["planes"], case["batch"], case["hkv"], n, case["dim"]), dtype=BF, device=DEV)
    for b, first in enumerate(s["row0"].tolist()):
        for k, page in enumerate(s["table"][b].tolist()):
            i, j = max(first, k * R), min(first + n, (k + 1) * R)  # the page's rows among them
            if i < j and case["op"] == "write":
                pool[:, page, :, i - k * R:j - k * R] = rows[:, b, :, i - first:j - first]
            elif i < j:
                rows[:, b, :, i - first:j - first] = pool[:, page, :, i - k * R:j - k * R]
    return [pool if case["op"] == "write" else rows]


def exact(case: dict, seed: int):
    """Attention in 64 bits; the other operators move rows, whose values stay what they are."""
    return {"tree": _exact_tree, "commit": _exact_commit, "fork": _exact_fork, "compact": _exact_compact,
            "write": _exact_rows, "read": _exact_rows}[case["op"]](_inputs(case, seed), case)
