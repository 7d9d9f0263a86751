"""Rotary positions, attention with modified scores and decode over a shared prefix, as measured calls.

Each case is one call as a generation program issues it, on inputs that are already on the GPU.
``run`` computes it in elementary torch operations in 32 bits, or, where ``own`` is true, through
the library.  Head shapes are this repository's (head_dim 128, 256, 512; GQA 2 to 8; one K = V
buffer at head_dim 512), with its 1024-token window.

Operators
  rope            rotary positions of the q and k rows of some tokens
  scored_decode   one decode step whose scores are capped by a tanh or biased by distance
  scored_prefill  a chunk's attention with a cap, a distance bias, a document or a prefix mask
  prefix          one decode step of a batch whose sequences share their first tokens
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
        # the new token of one user on a wide-head layer: the smallest call, latency only
        {"name": "rope_token", "op": "rope", "tokens": 1, "hq": 32, "hk": 4, "dim": 512, "rot": 512,
         "interleaved": False, "far": 131071, "scaling": "none", "inverse": False},
        # a long prompt, frequencies scaled in bands
        {"name": "rope_prompt_8k", "op": "rope", "tokens": 8192, "hq": 32, "hk": 8, "dim": 128, "rot": 128,
         "interleaved": False, "far": 8192, "scaling": "bands", "inverse": False},
        # a chunk far into a context, a quarter of each head rotated in interleaved pairs
        {"name": "rope_part_interleaved", "op": "rope", "tokens": 2049, "hq": 32, "hk": 16, "dim": 256, "rot": 64,
         "interleaved": True, "far": 1000003, "scaling": "yarn", "inverse": False},
        # a sliding layer with capped scores, one user: latency
        {"name": "capped_local_b1", "op": "scored_decode", "batch": 1, "hq": 16, "hkv": 8, "dim": 256, "cap": 1024,
         "ring": True, "softcap": 50.0, "biased": False},
        # a serving batch of ragged lengths with a bias per head instead of positions in q and k
        {"name": "biased_b16", "op": "scored_decode", "batch": 16, "hq": 32, "hkv": 8, "dim": 128, "cap": 16384,
         "ring": False, "softcap": 0.0, "biased": True},
        # a chunk of a long prompt over a capped K = V layer: the largest call
        {"name": "capped_chunk_16k", "op": "scored_prefill", "hq": 32, "hkv": 4, "dim": 512, "queries": 512,
         "past": 15872, "window": 0, "softcap": 30.0, "biased": False, "packed": False, "prefix": 0},
        # short documents packed into one row of 4096 tokens, the end of it padding
        {"name": "packed_documents_4k", "op": "scored_prefill", "hq": 32, "hkv": 8, "dim": 128, "queries": 4096,
         "past": 0, "window": 0, "softcap": 0.0, "biased": True, "packed": True, "prefix": 0},
        # a fresh prompt whose first 700 tokens see each other (an image, an instruction), sliding layer
        {"name": "prefix_mask_prompt", "op": "scored_prefill", "hq": 32, "hkv": 16, "dim": 256, "queries": 1511,
         "past": 0, "window": WINDOW, "softcap": 50.0, "biased": False, "packed": False, "prefix": 700},
        # two users behind one system prompt on a K = V layer
        {"name": "shared_b2", "op": "prefix", "batch": 2, "hq": 32, "hkv": 4, "dim": 512, "prefix": 2049, "cap": 256},
        # four samples of one long document on a K = V layer
        {"name": "shared_b4_32k", "op": "prefix", "batch": 4, "hq": 32, "hkv": 4, "dim": 512, "prefix": 32768,
         "cap": 512},
        # a serving batch behind one long instruction, head_dim 256
        {"name": "shared_b32", "op": "prefix", "batch": 32, "hq": 32, "hkv": 16, "dim": 256, "prefix": 8191,
         "cap": 512},
        # many samples of one prompt, head_dim 128
        {"name": "shared_b64", "op": "prefix", "batch": 64, "hq": 32, "hkv": 8, "dim": 128, "prefix": 16384,
         "cap": 1024},
    ]


def _log_uniform(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng) -> dict:
    op = rng.choice(["rope", "scored_decode", "scored_prefill", "scored_prefill", "prefix", "prefix"])
    if op == "rope":
        hq, hk = rng.choice([(32, 4), (32, 8), (32, 16), (16, 8)])
        dim = rng.choice([128, 256, 512])
        return {"op": op, "tokens": _log_uniform(rng, 1, 8192 * 128 // dim), "hq": hq, "hk": hk, "dim": dim,
                "rot": rng.choice([dim, dim, dim // 2, dim // 4, 40]), "interleaved": rng.random() < 0.5,
                "far": _log_uniform(rng, 8192, 2000000), "scaling": rng.choice(["none", "linear", "bands", "yarn"]),
                "inverse": rng.random() < 0.25}
    dim = rng.choice([128, 256, 512])
    hq, hkv = {128: rng.choice([(32, 8), (16, 8)]), 256: rng.choice([(32, 16), (16, 8)]),
               512: rng.choice([(32, 4), (16, 2)])}[dim]
    softcap, biased = rng.choice([(0.0, True), (20.0, True), (30.0, False), (50.0, False)])
    if op == "scored_decode":
        ring = rng.random() < 0.4
        batch = _log_uniform(rng, 1, 32)
        return {"op": op, "batch": batch, "hq": hq, "hkv": hkv, "dim": dim,
                "cap": WINDOW if ring else _log_uniform(rng, 64, 131072 // max(8, batch) * 2), "ring": ring,
                "softcap": softcap, "biased": biased}
    if op == "scored_prefill":
        packed = rng.random() < 0.4
        queries = _log_uniform(rng, 2, 4096 if dim == 128 else 2048)
        past = 0 if packed or queries > 512 else rng.choice([0, _log_uniform(rng, 64, 12000)])
        return {"op": op, "hq": hq, "hkv": hkv, "dim": dim, "queries": queries, "past": past,
                "window": rng.choice([0, 0, WINDOW]), "softcap": softcap, "biased": biased, "packed": packed,
                "prefix": 0 if past or rng.random() < 0.6 else _log_uniform(rng, 1, queries)}
    batch = _log_uniform(rng, 1, 64)
    return {"op": op, "batch": batch, "hq": hq, "hkv": hkv, "dim": dim,
            "prefix": _log_uniform(rng, 16, 16384 if batch > 8 else 49152), "cap": _log_uniform(rng, 16, 1024)}


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


def _frequencies(rot: int, scaling: str) -> tuple[torch.Tensor, float]:
    """Rotary inverse frequencies of base 10000 (a model's constants) and the factor on cos and sin."""
    half = rot // 2
    f = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device=DEV) * 2 / rot)
    factor, window = 8.0, 8192.0
    if scaling == "linear":
        return (f / factor).float(), 1.0
    if scaling == "none":
        return f.float(), 1.0
    turns = window * f / (2 * math.pi)  # over the trained window
    lo, hi = (1.0, 4.0) if scaling == "bands" else (1.0, 32.0)
    keep = ((turns - lo) / (hi - lo)).clamp(0.0, 1.0)
    scaled = keep * f + (1.0 - keep) * f / factor
    return scaled.float(), 1.0 if scaling == "bands" else 0.1 * math.log(factor) + 1.0


def _slopes(hq: int) -> torch.Tensor:
    """A geometric series of one slope per head, 2^-0.25 .. 2^-8."""
    return 2.0 ** (-8.0 * (torch.arange(hq, device=DEV, dtype=torch.float32) + 1) / hq)


def _rope_inputs(case: dict, g) -> dict:
    n, d = case["tokens"], case["dim"]
    start = case["far"] - n if case["far"] >= n else 0
    inv, factor = _frequencies(case["rot"], case["scaling"])
    return {"q": _rms_rows((n, case["hq"], d), g), "k": _rms_rows((n, case["hk"], d), g), "inv": inv, "factor": factor,
            "pos": start + torch.arange(n, device=DEV, dtype=torch.int32)}


def _lengths(batch: int, low: int, high: int, g) -> torch.Tensor:
    """Ragged lengths low .. high, the first one the longest."""
    n = torch.randint(low, high + 1, (batch,), device=DEV, generator=g, dtype=torch.int32)
    n[0] = high
    return n


def _decode_inputs(case: dict, g) -> dict:
    B, hq, hkv, d, cap = (case[x] for x in ("batch", "hq", "hkv", "dim", "cap"))
    s = {"q": _rms_rows((B, hq, d), g, 2.5), "k": _rms_rows((B, hkv, cap, d), g), "k_new": _rms_rows((B, hkv, d), g)}
    if d != 512:
        s["v"], s["v_new"] = _rms_rows((B, hkv, cap, d), g), _rms_rows((B, hkv, d), g)
    most = 32768 if case["ring"] else cap
    s["pos"] = _lengths(B, WINDOW if case["ring"] else max(1, cap // 8), most, g) - 1
    s["slopes"] = _slopes(hq) if case["biased"] else None
    return s


def _documents(n: int, g) -> torch.Tensor:
    """Ids of documents of 16 to about 1000 tokens packed one behind another; the last thirtieth is padding (-1)."""
    sizes = torch.exp(torch.rand(n // 16 + 1, device=DEV, generator=g) * math.log(1000 / 16)) * 16
    ends = sizes.long().cumsum(0)
    ids = torch.searchsorted(ends, torch.arange(n, device=DEV), right=True)
    return torch.where(torch.arange(n, device=DEV) < n - n // 30, ids, -1).to(torch.int32)


def _prefill_inputs(case: dict, g) -> dict:
    hq, hkv, d, n, past = (case[x] for x in ("hq", "hkv", "dim", "queries", "past"))
    first = max(0, past - case["window"] + 1) if case["window"] else 0  # a sliding layer keeps its window
    s = {"k_pos0": first, "q": _rms_rows((hq, n, d), g, 2.5), "k": _rms_rows((hkv, past + n - first, d), g)}
    s["v"] = s["k"] if d == 512 else _rms_rows((hkv, past + n - first, d), g)
    s["slopes"] = _slopes(hq) if case["biased"] else None
    s["doc"] = _documents(n, g) if case["packed"] else None
    return s


def _prefix_inputs(case: dict, g) -> dict:
    B, hq, hkv, d, P, cap = (case[x] for x in ("batch", "hq", "hkv", "dim", "prefix", "cap"))
    s = {"q": _rms_rows((B, hq, d), g, 2.0), "pk": _rms_rows((hkv, P, d), g), "k": _rms_rows((B, hkv, cap, d), g),
         "k_new": _rms_rows((B, hkv, d), g), "pos": P + _lengths(B, 1, cap, g) - 1}
    if d != 512:
        s["pv"], s["v"], s["v_new"] = (_rms_rows((hkv, P, d), g), _rms_rows((B, hkv, cap, d), g),
                                       _rms_rows((B, hkv, d), g))
    return s


def _inputs(case: dict, seed: int) -> dict:
    make = {"rope": _rope_inputs, "scored_decode": _decode_inputs, "scored_prefill": _prefill_inputs,
            "prefix": _prefix_inputs}[case["op"]]
    return make(case, _gen(seed))


def prepare(case: dict, seed: int) -> dict:
    return {"case": case, **_inputs(case, seed)}


# ------------------------------------------------------------------------------ plain forms

def _rotate(x: torch.Tensor, c: torch.Tensor, s: torch.Tensor, interleaved: bool) -> torch.Tensor:
    """x [tokens, heads, dim] turned by c, s [tokens, 1, pairs]; dims past the pairs stay."""
    r = 2 * c.shape[-1]
    xf = x.float()
    a, b = (xf[..., 0:r:2], xf[..., 1:r:2]) if interleaved else (xf[..., :r // 2], xf[..., r // 2:r])
    y0, y1 = a * c - b * s, b * c + a * s
    turned = torch.stack([y0, y1], dim=-1).flatten(-2) if interleaved else torch.cat([y0, y1], dim=-1)
    return torch.cat([turned, xf[..., r:]], dim=-1).to(BF)


def _plain_rope(st: dict):
    a = st["pos"].double().view(-1, 1, 1) * st["inv"].double()
    c = (st["factor"] * a.cos()).float()
    s = (st["factor"] * a.sin() * (-1.0 if st["case"]["inverse"] else 1.0)).float()
    return [_rotate(st["q"], c, s, st["case"]["interleaved"]), _rotate(st["k"], c, s, st["case"]["interleaved"])]


def _softmax_v(scores: torch.Tensor, hidden: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
    """Scores [.., q, k] float32, hidden entries left out, times v [.., k, d]; 0 for a row that sees nothing."""
    scores = scores.masked_fill(hidden, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = (scores - torch.where(torch.isinf(top), 0.0, top)).exp()
    total = p.sum(-1, keepdim=True)
    return (p @ v) / torch.where(total == 0, 1.0, total)


def _modified(scores: torch.Tensor, softcap: float) -> torch.Tensor:
    return softcap * torch.tanh(scores / softcap) if softcap else scores


def _append(cache: torch.Tensor, new: torch.Tensor, row: torch.Tensor) -> None:
    cache[torch.arange(cache.shape[0], device=DEV), :, row.long()] = new


def _plain_scored_decode(st: dict):
    case = st["case"]
    B, hq, hkv, d, cap = (case[x] for x in ("batch", "hq", "hkv", "dim", "cap"))
    pos = st["pos"].long()
    row = pos % cap if case["ring"] else pos
    _append(st["k"], st["k_new"], row)
    if d != 512:
        _append(st["v"], st["v_new"], row)
    kf = st["k"].float()
    vf = kf if d == 512 else st["v"].float()
    rows = torch.arange(cap, device=DEV)
    # how far behind the token the position in each row lies
    dist = ((row.unsqueeze(1) - rows) % cap if case["ring"] else pos.unsqueeze(1) - rows).view(B, 1, 1, cap)
    s = _modified(st["q"].float().view(B, hkv, hq // hkv, d) @ kf.transpose(-1, -2) * d ** -0.5, case["softcap"])
    if st["slopes"] is not None:
        s = s - st["slopes"].view(1, hkv, hq // hkv, 1) * dist
    hidden = (dist < 0) | (dist > pos.view(B, 1, 1, 1))
    out = _softmax_v(s, hidden, vf).reshape(B, hq, d).to(BF)
    return [out, st["k"]] + ([st["v"]] if d != 512 else [])


def _plain_scored_prefill(st: dict):
    case = st["case"]
    hq, hkv, d, n = (case[x] for x in ("hq", "hkv", "dim", "queries"))
    kf = st["k"].float()
    vf = kf if d == 512 else st["v"].float()
    q_at = (case["past"] + torch.arange(n, device=DEV)).unsqueeze(1)
    k_at = (st["k_pos0"] + torch.arange(kf.shape[1], device=DEV)).unsqueeze(0)
    hidden = (k_at > q_at) & (k_at >= case["prefix"])
    if case["window"]:
        hidden = hidden | (k_at <= q_at - case["window"])
    if st["doc"] is not None:
        ids = st["doc"]
        hidden = hidden | (ids.unsqueeze(1) != ids) | (ids < 0)
    qf = st["q"].float().reshape(hkv, hq // hkv * n, d)
    s = _modified((qf @ kf.transpose(-1, -2) * d ** -0.5).view(hkv, hq // hkv, n, -1), case["softcap"])
    if st["slopes"] is not None:
        s = s - st["slopes"].view(hkv, hq // hkv, 1, 1) * (q_at - k_at).abs()
    out = _softmax_v(s, hidden, vf.unsqueeze(1))
    return out.view(hq, n, d).transpose(0, 1).contiguous().to(BF)


def _plain_prefix(st: dict):
    case = st["case"]
    B, hq, hkv, d, P, cap = (case[x] for x in ("batch", "hq", "hkv", "dim", "prefix", "cap"))
    row = st["pos"].long() - P
    _append(st["k"], st["k_new"], row)
    if d != 512:
        _append(st["v"], st["v_new"], row)
    pk, kf = st["pk"].float(), st["k"].float()
    pv, vf = (pk, kf) if d == 512 else (st["pv"].float(), st["v"].float())
    q = st["q"].float().view(B, hkv, hq // hkv, d) * d ** -0.5
    G = hq // hkv
    shared = (q.transpose(0, 1).reshape(hkv, B * G, d) @ pk.transpose(-1, -2)).view(hkv, B, G, P).transpose(0, 1)
    tail = (q @ kf.transpose(-1, -2)).masked_fill(torch.arange(cap, device=DEV) > row.view(B, 1, 1, 1), -math.inf)
    top = torch.maximum(shared.amax(-1, keepdim=True), tail.amax(-1, keepdim=True))
    p, t = (shared - top).exp(), (tail - top).exp()
    o = (p.transpose(0, 1).reshape(hkv, B * G, P) @ pv).view(hkv, B, G, d).transpose(0, 1) + t @ vf
    out = (o / (p.sum(-1, keepdim=True) + t.sum(-1, keepdim=True))).reshape(B, hq, d).to(BF)
    return [out, st["k"]] + ([st["v"]] if d != 512 else [])


# ------------------------------------------------------------------------------ the library's calls

def _own_rope(st: dict):
    from apertura_amd.rope import RopeCall

    if "call" not in st:  # buffers and marshalled arguments, kept over a model's layers
        st["call"] = RopeCall(st["q"], st["k"], st["pos"], st["inv"], interleaved=st["case"]["interleaved"],
                              inverse=st["case"]["inverse"], attn_factor=st["factor"],
                              q_out=torch.empty_like(st["q"]), k_out=torch.empty_like(st["k"]))
    return list(st["call"]())


def _own_scored_decode(st: dict):
    from apertura_amd.decode import DecodeStep
    from apertura_amd.scored import Score, ScoredDecodeCall

    case = st["case"]
    if "call" not in st:
        step = DecodeStep.for_cache(st["k"], case["hq"], window=WINDOW if case["ring"] else 0, ring=case["ring"],
                                    kv_shared=case["dim"] == 512, scale=case["dim"] ** -0.5)
        st["call"] = ScoredDecodeCall(step, Score(softcap=case["softcap"], slopes=st["slopes"]), st["q"], st["k_new"],
                                      st.get("v_new"), st["k"], st.get("v", st["k"]), st["pos"])
    return [st["call"](), st["k"]] + ([st["v"]] if case["dim"] != 512 else [])


def _own_scored_prefill(st: dict):
    from apertura_amd.prefill import PrefillStep
    from apertura_amd.scored import Score, scored_prefill, scored_prefill_workspace_bytes

    case = st["case"]
    if "step" not in st:
        st["step"] = PrefillStep.for_tensors(st["q"], st["k"], q_pos0=case["past"], k_pos0=st["k_pos0"],
                                             window=case["window"], scale=case["dim"] ** -0.5)
        st["score"] = Score(softcap=case["softcap"], slopes=st["slopes"], prefix=case["prefix"])
        n = scored_prefill_workspace_bytes(st["step"], st["score"])
        st["workspace"] = torch.empty(n, dtype=torch.uint8, device=DEV) if n else None
    return scored_prefill(st["step"], st["score"], st["q"], st["k"], st["v"], q_doc=st["doc"], k_doc=st["doc"],
                          workspace=st["workspace"])


def _own_prefix(st: dict):
    from apertura_amd.prefix import PrefixCall, PrefixStep

    case = st["case"]
    if "call" not in st:
        step = PrefixStep.for_caches(st["pk"], st["k"], case["hq"], kv_shared=case["dim"] == 512,
                                     scale=case["dim"] ** -0.5)
        st["call"] = PrefixCall(step, st["q"], st["k_new"], st.get("v_new"), st["pk"], st.get("pv", st["pk"]), st["k"],
                                st.get("v", st["k"]), st["pos"])
    return [st["call"](), st["k"]] + ([st["v"]] if case["dim"] != 512 else [])


def run(st: dict):
    op = st["case"]["op"]
    if own:
        return {"rope": _own_rope, "scored_decode": _own_scored_decode, "scored_prefill": _own_scored_prefill,
                "prefix": _own_prefix}[op](st)
    return {"rope": _plain_rope, "scored_decode": _plain_scored_decode, "scored_prefill": _plain_scored_prefill,
            "prefix": _plain_prefix}[op](st)


# ------------------------------------------------------------------------------ work

def work(case: dict) -> dict:
    d = case["dim"]
    if case["op"] == "rope":
        heads = case["hq"] + case["hk"]
        return {"bytes": case["tokens"] * (4.0 * heads * d + 4) + 2 * case["rot"],
                "flops": 3.0 * case["tokens"] * heads * case["rot"]}
    hq, hkv = case["hq"], case["hkv"]
    streams = 1 if d == 512 else 2
    if case["op"] == "scored_prefill":
        n, past, w = case["queries"], case["past"], case["window"]
        pairs = 0
        for i in range(n):
            top = max(past + i + 1, min(case["prefix"], past + n))
            pairs += top - (max(0, past + i + 1 - w) if w else 0)
        if case["packed"]:  # the drawn documents' mean: 254 keys at or before a token, in its document
            pairs = min(pairs, 254 * (n - n // 30))
        keys = past + n - (max(0, past - w + 1) if w else 0)
        return {"bytes": 4.0 * n * hq * d + 2.0 * streams * hkv * keys * d, "flops": 4.0 * d * hq * pairs}
    B, cap = case["batch"], case["cap"]
    if case["op"] == "scored_decode":
        low = WINDOW if case["ring"] else max(1, cap // 8)
        rows = B * WINDOW if case["ring"] else cap + (B - 1) * (low + cap) // 2  # the mean of what is drawn
        products = rows * hq
        prefix = 0
    else:
        rows = cap + (B - 1) * (1 + cap) // 2
        prefix = case["prefix"]
        products = (rows + B * prefix) * hq
    return {"bytes": 2.0 * streams * hkv * d * (rows + prefix + B) + 4.0 * B * hq * d, "flops": 4.0 * d * products}


# ------------------------------------------------------------------------------ 64 bits

def _exact_rope(s: dict, case: dict) -> list:
    half = case["rot"] // 2
    sign = -1.0 if case["inverse"] else 1.0
    first = torch.arange(half, device=DEV)
    i, j = (2 * first, 2 * first + 1) if case["interleaved"] else (first, first + half)
    angle = s["pos"].double()[:, None] * s["inv"].double()[None]
    turn = torch.polar(torch.full_like(angle, s["factor"]), sign * angle)[:, None]
    outs = []
    for x in (s["q"], s["k"]):
        y = x.double()
        z = torch.complex(y[..., i], y[..., j]) * turn
        y[..., i], y[..., j] = z.real, z.imag
        outs.append(y)
    return outs


def _soft64(logits: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
    return torch.softmax(logits, dim=-1) @ v


def _cap64(x: torch.Tensor, softcap: float) -> torch.Tensor:
    return x if softcap == 0 else torch.tanh(x / softcap) * softcap


def _exact_decode(s: dict, case: dict) -> list:
    hq, hkv, d, cap = case["hq"], case["hkv"], case["dim"], case["cap"]
    G = hq // hkv
    out = torch.empty((case["batch"], hq, d), dtype=torch.float64, device=DEV)
    for b, p in enumerate(s["pos"].tolist()):
        seen = torch.arange(max(0, p + 1 - cap) if case["ring"] else 0, p + 1, device=DEV)
        k = s["k"][b][:, seen % cap].double()
        k[:, -1] = s["k_new"][b].double()
        v = k
        if d != 512:
            v = s["v"][b][:, seen % cap].double()
            v[:, -1] = s["v_new"][b].double()
        for h in range(hkv):
            x = _cap64(s["q"][b, h * G:(h + 1) * G].double() @ k[h].T / math.sqrt(d), case["softcap"])
            if case["biased"]:
                x = x - s["slopes"][h * G:(h + 1) * G, None].double() * (p - seen).double()
            out[b, h * G:(h + 1) * G] = _soft64(x, v[h])
    return [out, None] + ([None] if d != 512 else [])


def _exact_prefill(s: dict, case: dict) -> torch.Tensor:
    hq, hkv, d, n = case["hq"], case["hkv"], case["dim"], case["queries"]
    keys = s["k"].shape[1]
    gap = (case["past"] + torch.arange(n, device=DEV))[:, None] - (s["k_pos0"] + torch.arange(keys, device=DEV))[None]
    seen = (gap >= 0) | ((s["k_pos0"] + torch.arange(keys, device=DEV)) < case["prefix"])[None]
    if case["window"]:
        seen = seen & (gap < case["window"])
    if case["packed"]:
        ids = s["doc"]
        seen = seen & (ids[:, None] == ids[None]) & (ids >= 0)[:, None]
    out = torch.empty((n, hq, d), dtype=torch.float64, device=DEV)
    for h in range(hq):
        kvh = h // (hq // hkv)
        x = _cap64(s["q"][h].double() @ s["k"][kvh].double().T / math.sqrt(d), case["softcap"])
        if case["biased"]:
            x = x - s["slopes"][h].double() * gap.abs().double()
        w = torch.nan_to_num(torch.softmax(torch.where(seen, x, -math.inf), dim=-1))
        out[:, h] = w @ s["v"][kvh].double()
    return out


def _exact_prefix(s: dict, case: dict) -> list:
    hq, hkv, d, P = case["hq"], case["hkv"], case["dim"], case["prefix"]
    G = hq // hkv
    out = torch.empty((case["batch"], hq, d), dtype=torch.float64, device=DEV)
    for b, p in enumerate(s["pos"].tolist()):
        m = p - P
        k = torch.cat([s["pk"], s["k"][b, :, :m], s["k_new"][b][:, None]], dim=1).double()
        v = k
        if d != 512:
            v = torch.cat([s["pv"], s["v"][b, :, :m], s["v_new"][b][:, None]], dim=1).double()
        x = s["q"][b].double().view(hkv, G, d) @ k.transpose(1, 2) / math.sqrt(d)
        out[b] = _soft64(x, v).reshape(hq, d)
    return [out, None] + ([None] if d != 512 else [])


def exact(case: dict, seed: int):
    s = _inputs(case, seed)
    return {"rope": _exact_rope, "scored_decode": _exact_decode, "scored_prefill": _exact_prefill,
            "prefix": _exact_prefix}[case["op"]](s, case)
