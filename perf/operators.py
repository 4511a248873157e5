"""Operators on rows held in 8 bits and on beams, timed in their plain form and through the library.

One step of a generating model that keeps its weights and rows in 8 bits: the residual's addition, the norm and the row's codes; the
product of codes; the selection over beams and vocabulary; the states brought into the new beams' order.  The same product scores
stored 8-bit rows against queries.

  encode   rows to 8-bit codes, one scale a row
  norm     residual addition, root-mean-square norm, 8-bit codes with one scale a row
  matmul   products of 8-bit codes with the scales of rows (tokens, queries) and columns (channels, stored rows)
  select   the best continuations of every batch item over its beams and the vocabulary
  reorder  states (keys, values) brought into the order of the chosen beams

Codes are whole numbers: code = rint(127 u / max|u|) with ties to even is settled in 64 bits wherever 32 bits leave it open, so
they have to be equal.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # stored rows of the benchmark's large index dimension, brought to 8 bits when an index is built
        dict(name="encode_stored", kind="encode", n=1_000_000, dim=96, type="f32", pad=0),
        # a few activations of an odd width in a padded buffer whose rows begin at odd places
        dict(name="encode_odd", kind="encode", n=333, dim=5003, type="f16", pad=9),
        # one token of a decoding step: latency is all
        dict(name="norm_token", kind="norm", n=1, dim=4096, type="bf16", residual=True),
        # a prompt's tokens
        dict(name="norm_prompt", kind="norm", n=16_384, dim=8192, type="bf16", residual=True),
        # one token's logits: the whole vocabulary matrix is read for one row
        dict(name="matmul_token", kind="matmul", m=1, n=32_000, k=4096, type="bf16"),
        # a small batch, nothing a multiple of a tile, a layer too narrow to fill the GPU with one tile a block
        dict(name="matmul_odd", kind="matmul", m=37, n=4099, k=4000, type="f16"),
        # a prompt through a wide layer: the tensor cores' rate
        dict(name="matmul_prompt", kind="matmul", m=8192, n=8192, k=8192, type="bf16"),
        # queries against stored 8-bit rows, all scores wanted: short products, the scores' writes are what counts
        dict(name="matmul_scores", kind="matmul", m=100, n=500_000, k=128, type="f32"),
        # one sequence's beam search step: latency
        dict(name="select_one", kind="select", batch=1, beams=4, vocab=32_000, k=8, type="f32", pad=0),
        # a serving batch with a large vocabulary
        dict(name="select_batch", kind="select", batch=64, beams=8, vocab=128_000, k=16, type="bf16", pad=0),
        # a step's reordering in place, sequences of different lengths, the surviving beams keep their slots
        dict(name="reorder_place", kind="reorder", layers=2, batch=5, beams=4, heads=8, tokens=515, dim=64, type="f16", place=True),
        # long sequences into a second buffer, every beam moves
        dict(name="reorder_long", kind="reorder", layers=4, batch=16, beams=4, heads=8, tokens=2048, dim=128, type="bf16", place=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["encode", "norm", "matmul", "select", "reorder"])
    kind_type = rng.choice(["f32", "f16", "bf16"])
    if kind == "encode":
        dim = _log(rng, 16, 20_000)
        return dict(kind=kind, n=_log(rng, 1, min(1_000_000, 90_000_000 // dim)), dim=dim, type=kind_type, pad=rng.choice([0, 0, 3, 16]))
    if kind == "norm":
        dim = _log(rng, 64, 16_384)
        return dict(kind=kind, n=_log(rng, 1, min(100_000, 60_000_000 // dim)), dim=dim, type=kind_type, residual=rng.random() < 0.7)
    if kind == "matmul":
        m, k = _log(rng, 1, 8192), _log(rng, 64, 16_384)
        n = _log(rng, 64, min(200_000, 250_000_000_000 // (m * k), 50_000_000 // m, 500_000_000 // k))
        return dict(kind=kind, m=m, n=n, k=k, type=kind_type)
    if kind == "select":
        beams, vocab = rng.randint(1, 16), _log(rng, 500, 200_000)
        batch = _log(rng, 1, min(128, max(1, 40_000_000 // (beams * vocab))))
        return dict(kind=kind, batch=batch, beams=beams, vocab=vocab, k=rng.randint(1, 2 * beams), type=kind_type, pad=rng.choice([0, 0, 1, 8]))
    beams, tokens, dim, place = rng.randint(2, 8), _log(rng, 1, 4096), rng.choice([64, 80, 128, 256]), rng.random() < 0.5
    batch = _log(rng, 1, min(32, max(1, 30_000_000 // (16 * beams * tokens * dim))))
    return dict(kind=kind, layers=2, batch=batch, beams=beams, heads=8, tokens=tokens, dim=dim, type=rng.choice(["f16", "bf16"]), place=place)


def _lengths(c):
    """Tokens of each batch item's sequences: up to a third shorter than the buffer."""
    return [max(1, c["tokens"] - (i * 37) % max(1, c["tokens"] // 3)) for i in range(c["batch"])]


def prepare(case, seed):
    c, kind = case, case["kind"]
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    s = dict(case)
    if kind in ("encode", "norm"):
        t, n, dim, pad = TYPES[c["type"]], c["n"], c["dim"], c.get("pad", 0)
        # rows of different magnitudes, a few channels far larger than the rest, as activations have them
        x = normal(n, dim + pad).mul_(torch.exp(normal(n, 1)))
        x[:, : max(1, dim // 128)] *= 8
        if n > 4:
            x[n // 2] = 0
        s["x"] = x.to(t)[:, :dim]
        s["codes"] = torch.empty((n, dim), dtype=torch.int8, device="cuda")
        s["scales"] = torch.empty(n, device="cuda")
        if kind == "norm":
            s["residual"] = normal(n, dim).to(t) if c["residual"] else None
            s["weight"] = (1 + 0.1 * normal(dim)).to(t)
            s["sum"] = torch.empty((n, dim), dtype=t, device="cuda") if c["residual"] else None
            s["eps"] = 1e-5
    elif kind == "matmul":
        m, n, k = c["m"], c["n"], c["k"]
        pitch = (k + 15) // 16 * 16   # rows begin at multiples of 16 bytes, as the library's encoders are asked to lay them out
        codes = lambda rows: normal(rows, pitch).mul_(40).round_().clamp_(-127, 127).to(torch.int8)[:, :k]  # noqa: E731
        s["x"], s["w"] = codes(m), codes(n)
        s["x_scales"] = torch.exp(normal(m)) / 40
        s["w_scales"] = torch.exp(0.2 * normal(n)) / (40 * math.sqrt(k))
        s["out"] = torch.empty((m, n), dtype=TYPES[c["type"]], device="cuda")
    elif kind == "select":
        rows, vocab, k = c["batch"] * c["beams"], c["vocab"], c["k"]
        x = normal(rows, vocab + c["pad"]).mul_(3)
        x[:, torch.randint(0, vocab, (max(1, vocab // 200),), generator=g, device="cuda")] = -math.inf   # tokens that are ruled out
        s["logits"] = x.to(TYPES[c["type"]])[:, :vocab]
        s["scores"] = -5 * torch.rand((c["batch"], c["beams"]), generator=g, device="cuda")
        if c["beams"] > 2:
            s["scores"][:, 1] = -math.inf   # a beam that has ended
        s["parents"] = torch.empty((c["batch"], k), dtype=torch.int32, device="cuda")
        s["tokens"] = torch.empty((c["batch"], k), dtype=torch.int32, device="cuda")
        s["totals"] = torch.empty((c["batch"], k), device="cuda")
    else:
        batch, beams = c["batch"], c["beams"]
        shape = (c["layers"], batch, beams, c["heads"], c["tokens"], c["dim"])
        s["states"] = torch.randn(shape, generator=g, device="cuda", dtype=TYPES[c["type"]])
        order = torch.rand((batch, beams), generator=g, device="cuda").argsort(1)
        keep = (beams + 1) // 2   # beams that live on
        parents = order[:, torch.arange(beams, device="cuda") % keep]
        if c["place"]:   # they keep their slots, the others' slots take copies: a second pass leaves things as they are
            s["parents"] = torch.empty_like(parents).scatter_(1, order, parents).int()
        else:
            s["parents"] = parents.int()
            s["out"] = torch.zeros_like(s["states"])
        s["lengths"] = torch.tensor(_lengths(c), dtype=torch.int32, device="cuda")
    return s


def _codes(u):
    """Codes and the largest magnitude of each row, from values in 64 bits."""
    top = u.abs().amax(1, keepdim=True)
    return torch.where(top > 0, 127 * u / top, 0.0).round_().to(torch.int8), top[:, 0]


def _plain(s):
    kind = s["kind"]
    if kind == "encode":
        codes, top = _codes(s["x"].double())
        return {"codes": codes, "scales": top.float() / 127}
    if kind == "norm":
        h, u = s["x"].float(), s["x"].double()
        if s["residual"] is not None:
            h, u = h + s["residual"].float(), u + s["residual"].double()
        codes, top = _codes(u * s["weight"].double())
        inverse = torch.rsqrt(h.square().mean(1) + s["eps"])
        out = {"codes": codes, "scales": top.float() * inverse / 127}
        return out if s["residual"] is None else {**out, "sum": h.to(s["x"].dtype)}
    if kind == "matmul":
        p = s["x"].float() @ s["w"].float().T
        return {"out": (p * s["x_scales"][:, None] * s["w_scales"]).to(s["out"].dtype)}
    if kind == "select":
        batch, beams, vocab, k = s["batch"], s["beams"], s["vocab"], s["k"]
        x = s["logits"].reshape(batch, beams, vocab)
        top = x.amax(2, keepdim=True).double()
        log_sum = torch.exp(x.double() - top).sum(2, keepdim=True).log()
        few = min(k, vocab)
        value, token = (a[:, :, :few] for a in torch.sort(x, dim=2, descending=True, stable=True))
        start = s["scores"].double()[:, :, None]
        total = start + ((value.double() - top) - log_sum)
        total = torch.where(torch.isfinite(top) & torch.isfinite(log_sum) & torch.isfinite(start), total, -math.inf).reshape(batch, beams * few)
        total, at = (a[:, :k] for a in torch.sort(total, dim=1, descending=True, stable=True))
        none = total == -math.inf
        parents = torch.where(none, -1, at // few).int()
        tokens = torch.where(none, -1, token.reshape(batch, beams * few).gather(1, at)).int()
        return {"parents": parents, "tokens": tokens, "totals": total.float()}
    states, out = s["states"], s["states"] if s["place"] else s["out"]
    item = torch.arange(s["batch"], device="cuda")[:, None]
    moved = states[:, item, s["parents"].long()]
    live = (torch.arange(s["tokens"], device="cuda")[None, :] < s["lengths"][:, None])[None, :, None, None, :, None]
    out.copy_(torch.where(live, moved, out))
    return {"states": out}


def _own(s):
    from paraselect_b200 import api
    kind = s["kind"]
    if kind == "encode":
        api.i8_encode_rows(s["x"], s["n"], s["dim"], s["codes"], s["scales"], row_stride=s["x"].stride(0))
        return {"codes": s["codes"], "scales": s["scales"]}
    if kind == "norm":
        api.i8_norm_rows(s["x"], s["n"], s["dim"], s["weight"], s["eps"], s["codes"], s["scales"], d_residual=s["residual"], d_sum=s["sum"])
        out = {"codes": s["codes"], "scales": s["scales"]}
        return out if s["residual"] is None else {**out, "sum": s["sum"]}
    if kind == "matmul":
        api.i8_matmul(s["x"], s["x_scales"], s["m"], s["w"], s["w_scales"], s["n"], s["k"], s["out"],
                      x_stride=s["x"].stride(0), w_stride=s["w"].stride(0))
        return {"out": s["out"]}
    if kind == "select":
        api.beam_select(s["logits"], s["scores"], s["batch"], s["beams"], s["vocab"], s["k"], s["parents"], s["tokens"], s["totals"],
                        row_stride=s["logits"].stride(0))
        return {"parents": s["parents"], "tokens": s["tokens"], "totals": s["totals"]}
    states, out = s["states"], s["states"] if s["place"] else s["out"]
    token_bytes = s["dim"] * states.element_size()
    api.beam_reorder(states, out, s["parents"], s["layers"], s["batch"], s["beams"], s["heads"], s["tokens"], token_bytes,
                     d_lengths=s["lengths"])
    return {"states": out}


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    c, kind = case, case["kind"]
    if kind == "encode":
        n = c["n"] * c["dim"]
        return {"bytes": n * (SIZE[c["type"]] + 1) + 4 * c["n"], "flops": 4 * n}
    if kind == "norm":
        n, e = c["n"] * c["dim"], SIZE[c["type"]]
        return {"bytes": n * (e * (3 if c["residual"] else 1) + 1) + 4 * c["n"] + c["dim"] * e, "flops": 8 * n}
    if kind == "matmul":
        m, n, k = c["m"], c["n"], c["k"]
        return {"bytes": (m + n) * (k + 4) + m * n * SIZE[c["type"]], "flops": 2 * m * n * k}
    if kind == "select":
        n = c["batch"] * c["beams"] * c["vocab"]
        return {"bytes": n * SIZE[c["type"]] + 4 * c["batch"] * (c["beams"] + 3 * c["k"]), "flops": 4 * n}
    # rows (one layer's state of one beam) that have to be read and written
    keep = (c["beams"] + 1) // 2
    rows = min(keep, c["beams"] - keep) + c["beams"] - keep if c["place"] else keep + c["beams"]
    return {"bytes": c["layers"] * rows * sum(_lengths(c)) * c["heads"] * c["dim"] * SIZE[c["type"]], "flops": 0}


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind in ("encode", "norm"):
        h = s["x"].double()
        if kind == "norm" and s["residual"] is not None:
            h = h.add(s["residual"])
        u = h * s["weight"].double() if kind == "norm" else h
        top = torch.maximum(u.amax(1), -u.amin(1))
        codes = torch.round(127.0 * u / torch.where(top == 0, 1.0, top).unsqueeze(1)).to(torch.int8)
        if kind == "encode":
            return {"codes": codes, "scales": top / 127}
        rms = ((h * h).sum(1) / case["dim"] + s["eps"]).sqrt()
        out = {"codes": codes, "scales": top / (rms * 127)}
        return out if s["residual"] is None else {**out, "sum": h}
    if kind == "matmul":
        x, w = s["x"].double() * s["x_scales"].double()[:, None], s["w"].double() * s["w_scales"].double()[:, None]
        return {"out": torch.mm(x, w.t())}
    if kind == "select":
        batch, beams, vocab, k = case["batch"], case["beams"], case["vocab"], case["k"]
        p = torch.log_softmax(s["logits"].double(), 1).view(batch, beams, vocab) + s["scores"].double().unsqueeze(2)
        p = torch.where(p.isnan(), -math.inf, p).view(batch, beams * vocab)
        p, at = torch.sort(p, dim=1, descending=True, stable=True)
        p, at = p[:, :k], at[:, :k]
        if p.shape[1] < k:
            return None
        gone = torch.isneginf(p)
        return {"parents": (at // vocab).masked_fill(gone, -1).int(), "tokens": (at % vocab).masked_fill(gone, -1).int(), "totals": p}
    out = s["states"].clone() if case["place"] else s["out"]
    rows, parents = s["states"].clone(), s["parents"].tolist()
    for b, n in enumerate(_lengths(case)):
        for j, p in enumerate(parents[b]):
            out[:, b, j, :, :n] = rows[:, b, p, :, :n]
    return {"states": out}
