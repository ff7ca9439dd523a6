"""The operators at the end of a decode step and the calls that are measured of them:

  norm     the residual's addition, the root-mean-square norm, and its output in 8-bit
           integers with a scale for each token;
  product  the unembedding product in 8-bit integers, with a scale for each token and for
           each vocabulary entry (channel), to fp32 or bf16 logits;
  beam     beam search's selection over beams and vocabulary, with the reordering of the
           search's rows: penalty history rings and cached states.

``run`` computes each in elementary torch operations, or (``own``) through the public
Python interface of the library.
"""
import math

import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}
_INF = float("inf")


def listed():
    return [
        # One token of one sequence: what a single user's decode step waits for.
        {"name": "norm 1x2560 f32", "op": "norm", "rows": 1, "dim": 2560, "dtype": "f32", "residual": True},
        # A decode batch with an odd width.
        {"name": "norm 37x1001 f16", "op": "norm", "rows": 37, "dim": 1001, "dtype": "f16", "residual": False},
        # A prompt's tokens, as a prefill step passes them between layers.
        {"name": "norm 8192x3840 bf16", "op": "norm", "rows": 8192, "dim": 3840, "dtype": "bf16", "residual": True},
        # Logits of one sequence: the weights are read once.
        {"name": "product 1x1152x262144 f32", "op": "product", "batch": 1, "in_dim": 1152, "out_dim": 262144,
         "dtype": "f32"},
        # A ragged decode batch over a small vocabulary, the vocabulary not a multiple of anything.
        {"name": "product 37x3840x32003 bf16", "op": "product", "batch": 37, "in_dim": 3840, "out_dim": 32003,
         "dtype": "bf16"},
        # An ordinary serving batch.
        {"name": "product 64x2560x262144 f32", "op": "product", "batch": 64, "in_dim": 2560, "out_dim": 262144,
         "dtype": "f32"},
        # The largest batch the sampler is benchmarked with.
        {"name": "product 512x2560x262144 f32", "op": "product", "batch": 512, "in_dim": 2560, "out_dim": 262144,
         "dtype": "f32"},
        # One prompt's search over a small vocabulary: latency.
        {"name": "beam 1x4x32000 f32", "op": "beam", "batch": 1, "beams": 4, "vocab": 32000, "dtype": "f32",
         "window": 0, "penalty": 1.0, "alpha": 0.0, "heads": 0, "used": 0, "room": 0, "width": 0},
        # A few prompts, odd vocabulary, a repetition penalty and one layer's key and value cache to reorder.
        {"name": "beam 8x5x50257 bf16", "op": "beam", "batch": 8, "beams": 5, "vocab": 50257, "dtype": "bf16",
         "window": 64, "penalty": 1.1, "alpha": 0.6, "heads": 8, "used": 777, "room": 1024, "width": 128},
        # The library's vocabulary, a wide search.
        {"name": "beam 4x16x262144 bf16", "op": "beam", "batch": 4, "beams": 16, "vocab": 262144, "dtype": "bf16",
         "window": 64, "penalty": 1.2, "alpha": 1.0, "heads": 0, "used": 0, "room": 0, "width": 0},
        # Long sequences: the reordering of the cache outweighs the selection.
        {"name": "beam 16x4x32000 long cache", "op": "beam", "batch": 16, "beams": 4, "vocab": 32000, "dtype": "f32",
         "window": 512, "penalty": 1.1, "alpha": 0.0, "heads": 4, "used": 2500, "room": 2560, "width": 256},
        # The largest: 512 rows of logits, larger than L2.
        {"name": "beam 64x8x262144 f32", "op": "beam", "batch": 64, "beams": 8, "vocab": 262144, "dtype": "f32",
         "window": 0, "penalty": 1.0, "alpha": 0.0, "heads": 0, "used": 0, "room": 0, "width": 0},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "product", "beam"])
    if op == "norm":
        dim, dtype = _log_int(rng, 64, 8192), rng.choice(["f32", "bf16", "f16"])
        most = 8192 * 3840 * 7 // (dim * (3 * _SIZE[dtype] + 1))
        return {"op": "norm", "rows": _log_int(rng, 1, min(8192, most)), "dim": dim, "dtype": dtype,
                "residual": rng.random() < 0.7}
    if op == "product":
        in_dim = _log_int(rng, 64, 8192)
        out_dim = _log_int(rng, 1000, min(262144, 2560 * 262144 // in_dim))
        return {"op": "product", "batch": _log_int(rng, 1, 512), "in_dim": in_dim, "out_dim": out_dim,
                "dtype": rng.choice(["f32", "bf16"])}
    beams, vocab = rng.randint(1, 16), _log_int(rng, 1000, 262144)
    batch = _log_int(rng, 1, max(1, min(64, 512 * 262144 // (beams * vocab), 256 // beams)))
    window = rng.choice([0, 16, 64, 100])
    heads = rng.choice([0, 0, 1, 4, 8])
    used = _log_int(rng, 1, 1024) if heads else 0
    return {"op": "beam", "batch": batch, "beams": beams, "vocab": vocab, "dtype": rng.choice(["f32", "bf16"]),
            "window": window, "penalty": round(rng.uniform(1.05, 1.5), 2) if window else 1.0,
            "alpha": rng.choice([0.0, 0.6, 1.0]), "heads": heads, "used": used,
            "room": used + rng.randint(0, 300) if heads else 0, "width": rng.choice([64, 72, 128]) if heads else 0}


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)


def _randint(g, lo, hi, *shape, dtype=torch.int32):
    return torch.randint(lo, hi, shape, generator=g, device="cuda", dtype=dtype)


def _context():
    from vindexllm_b200.sampler import SamplerContext
    return SamplerContext(torch.cuda.current_device())


def prepare(case, seed):
    g, s = _gen(seed), {"case": case}
    if case["op"] == "norm":
        rows, dim, dt = case["rows"], case["dim"], _DT[case["dtype"]]
        # Hidden states: a few channels are much larger than the rest.
        channel = 1.0 + 20.0 * (torch.rand(dim, generator=g, device="cuda") < 0.005)
        s["x"] = (_randn(g, rows, dim) * channel).to(dt)
        s["residual"] = (_randn(g, rows, dim) * channel * 3.0).to(dt) if case["residual"] else None
        s["weight"] = 1.0 + 0.2 * _randn(g, dim)
        s["eps"] = 1e-6
        if own:
            s["ctx"] = _context()
    elif case["op"] == "product":
        batch, k, n = case["batch"], case["in_dim"], case["out_dim"]
        # Activations as the norm leaves them: rows padded to a multiple of 16 bytes.
        room = -(-k // 16) * 16
        s["q"] = (_randn(g, batch, room) * 32.0).round_().clamp_(-127, 127).to(torch.int8)[:, :k]
        s["q_scale"] = 0.01 + 0.05 * torch.rand(batch, generator=g, device="cuda")
        w = torch.empty(n, k, dtype=torch.int8, device="cuda")
        for at in range(0, n, 32768):
            part = w[at:at + 32768]
            part.copy_((_randn(g, *part.shape, dtype=torch.float16) * 36.0).round_().clamp_(-127, 127))
        w_scale = 0.0005 + 0.001 * torch.rand(n, generator=g, device="cuda")
        if own:
            from vindexllm_b200.sampler import I8Weights
            s["ctx"] = _context()
            s["weights"] = I8Weights(s["ctx"], w, w_scale)
        else:
            s["w"], s["w_scale"] = w, w_scale
    else:
        batch, beams, vocab, window = case["batch"], case["beams"], case["vocab"], case["window"]
        rows = batch * beams
        x = _randn(g, rows, vocab, dtype=torch.float32).mul_(3.0)
        peaks = _randint(g, 0, vocab, rows, 12, dtype=torch.int64)
        x.scatter_(1, peaks, 10.0 + 3.0 * _randn(g, rows, 12))
        s["logits"] = x.to(_DT[case["dtype"]])
        s["stop_ids"] = _randint(g, 0, vocab, 2)
        s["scores"] = -20.0 + 3.0 * _randn(g, rows)
        s["lengths"] = _randint(g, 5, 40, rows)
        s["finished"] = (torch.rand(rows, generator=g, device="cuda") < 0.15).to(torch.int32)
        if window:
            # Rings part filled, with tokens that the rows like and tokens that they do not.
            s["hist"] = _randint(g, 0, vocab, rows, window)
            s["hist"][:, :min(6, window)] = peaks[:, :min(6, window)].to(torch.int32)
            s["count"] = _randint(g, window // 2, window + 1, rows)
            s["pos"] = s["count"] % window
        if case["heads"]:
            shape = (rows, case["heads"], case["room"], case["width"])
            s["caches"] = [_randn(g, *shape, dtype=torch.bfloat16) for _ in range(2)]
            s["caches_out"] = [torch.zeros_like(c) for c in s["caches"]]
        if own:
            from vindexllm_b200.sampler import BeamSearch, BeamState
            s["ctx"] = _context()
            s["search"] = BeamSearch(s["ctx"], batch, beams, vocab)
            s["now"] = BeamState(batch, beams, window, scores=s["scores"], lengths=s["lengths"],
                                 finished=s["finished"], hist=s.get("hist"), pos=s.get("pos"), count=s.get("count"))
            s["next"] = BeamState(batch, beams, window)
    return s


def run(s):
    return {"norm": _norm, "product": _product, "beam": _beam}[s["case"]["op"]](s)


def _norm(s):
    """h = x + residual in the inputs' type; y = h * weight / sqrt(mean(h^2) + eps);
    scale = max|y| / 127, q = y / scale rounded to the nearest even integer."""
    if own:
        q, scale, h = s["ctx"].rms_norm_i8(s["x"], s["weight"], s["eps"], residual=s["residual"])
        return {"y": q * scale[:, None], "scale": scale, "h": h}
    h = s["x"]
    if s["residual"] is not None:
        h = (h.float() + s["residual"].float()).to(h.dtype)
    # 64 bits: a value next to a rounding border must fall on its own side.
    hd = h.double()
    t = hd * s["weight"].double()
    top = t.abs().amax(1, keepdim=True)
    q = torch.where(top > 0, torch.round(t * 127.0 / top), 0.0)
    scale = (top / 127.0 / torch.sqrt(hd.square().mean(1, keepdim=True) + s["eps"])).float()
    return {"y": q.float() * scale, "scale": scale[:, 0], "h": h if s["residual"] is not None else None}


def _product(s):
    """logits[b][n] = q_scale[b] * w_scale[n] * sum_k q[b][k] w[n][k]."""
    if own:
        return s["weights"].unembed(s["q"], s["q_scale"], dtype=_DT[s["case"]["dtype"]])
    y = s["q"].float() @ s["w"].float().T
    return y.mul_(s["w_scale"]).mul_(s["q_scale"][:, None]).to(_DT[s["case"]["dtype"]])


def _beam(s):
    """One step of the search for every prompt. A live beam b offers its `beams` largest
    logits v (equal ones by lower token) with the score s_b + log softmax(logits_b)[v] and the
    length n_b + 1; a finished beam offers itself, unchanged. The `beams` offers with the
    highest score / length^alpha stay (equal ones: lower beam, then the beam's own order)."""
    case = s["case"]
    batch, beams, vocab, window = case["batch"], case["beams"], case["vocab"], case["window"]
    rows, device = batch * beams, s["logits"].device
    if own:
        used = case["used"]
        caches = [(a[:, :, :used], b[:, :, :used]) for a, b in zip(s["caches"], s["caches_out"])] if case["heads"] else []
        tokens, parents = s["search"].step(s["now"], s["logits"], out=s["next"], stop_ids=s["stop_ids"], pad_token=0,
                                           repeat_penalty=case["penalty"], length_alpha=case["alpha"], caches=caches)
        n = s["next"]
        ring = [n.hist, n.pos, n.count] if window else None
        return {"tokens": tokens, "parents": parents, "scores": n.scores, "lengths": n.lengths,
                "finished": n.finished, "ring": ring, "caches": s["caches_out"] if case["heads"] else None}
    x = s["logits"].float()
    if window and case["penalty"] != 1.0:
        # x > 0: x / p, else x * p, once for each time that the ring holds the token.
        filled = torch.arange(window, device=device) < s["count"][:, None]
        times = torch.zeros(rows, vocab, device=device).scatter_add_(1, s["hist"].long(), filled.float())
        power = torch.pow(torch.tensor(case["penalty"], device=device).double(), times.double())
        x = torch.where(times > 0, torch.where(x > 0, x.double() / power, x.double() * power), x.double()).float()
    # 64 bits: offers of different beams are next to one another, and the sums are long.
    top = x.amax(1, keepdim=True).double()
    total = (top + torch.log(torch.exp(x.double() - top).sum(1, keepdim=True)))
    # The order of the values in whole numbers, with the lower token first among equals.
    bits = x.view(torch.int32).long()
    order = torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF)) * (1 << 32)
    order += (1 << 32) - 1 - torch.arange(vocab, device=device)
    n = min(beams, vocab)
    token = (1 << 32) - 1 - (torch.topk(order, n, dim=1).values & 0xFFFFFFFF)
    done = s["finished"][:, None] != 0
    before = s["scores"].double()[:, None]
    score = before + (x.gather(1, token).double() - total)
    first = torch.arange(n, device=device) == 0
    score = torch.where(done, torch.where(first, before, -_INF), score)
    token = torch.where(done, 0, token)
    length = (s["lengths"][:, None] + torch.where(done, 0, 1)).expand(rows, n)
    rank = torch.where(score > -_INF, score / length.double() ** case["alpha"], -_INF).reshape(batch, beams * n)
    pick = torch.sort(rank, dim=1, descending=True, stable=True).indices[:, :beams]
    kept = rank.gather(1, pick) > -_INF
    own_slot = torch.arange(beams, device=device).expand(batch, beams)
    parents = torch.where(kept, pick // n, own_slot)
    source = (parents + beams * torch.arange(batch, device=device)[:, None]).reshape(-1)

    def take(v):
        return v.reshape(batch, beams * n).gather(1, pick).reshape(-1)

    kept = kept.reshape(-1)
    tokens = torch.where(kept, take(token), 0)
    new = kept & (s["finished"][source] == 0)
    stop = (tokens[:, None] == s["stop_ids"]).any(1)
    scores = torch.where(kept, take(score).float(), -_INF)
    lengths = torch.where(kept, take(length), s["lengths"])
    finished = torch.where(kept, torch.where(new, stop, True), False)
    ring = None
    if window:
        at, held = s["pos"][source], s["count"][source]
        hit = new[:, None] & (torch.arange(window, device=device) == at[:, None])
        ring = [torch.where(hit, tokens[:, None], s["hist"][source].long()).int(),
                torch.where(new, (at + 1) % window, at).int(), torch.where(new, (held + 1).clamp(max=window), held).int()]
    if case["heads"]:
        torch._foreach_copy_([c[:, :, :case["used"]] for c in s["caches_out"]],
                             [c[source, :, :case["used"]] for c in s["caches"]])
    return {"tokens": tokens.int().view(batch, beams), "parents": parents.int(), "scores": scores,
            "lengths": lengths.int(), "finished": finished.int(), "ring": ring,
            "caches": s["caches_out"] if case["heads"] else None}


def work(case):
    if case["op"] == "norm":
        n, b = case["rows"] * case["dim"], _SIZE[case["dtype"]]
        return {"bytes": n * (b * (3 if case["residual"] else 1) + 1) + 4 * (case["dim"] + case["rows"]),
                "flops": 6 * n}
    if case["op"] == "product":
        b, k, n = case["batch"], case["in_dim"], case["out_dim"]
        return {"bytes": n * k + b * k + 4 * (n + b) + b * n * _SIZE[case["dtype"]], "flops": 2 * b * k * n}
    rows = case["batch"] * case["beams"]
    logits = rows * case["vocab"]
    moved = rows * (case["window"] * 4 + 2 * case["heads"] * case["used"] * case["width"] * 2 + 20)
    return {"bytes": logits * _SIZE[case["dtype"]] + 2 * moved, "flops": 4 * logits}


def exact(case, seed):
    global own
    before, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = before
    if case["op"] == "norm":
        h = s["x"].double()
        if s["residual"] is not None:
            h = torch.add(h, s["residual"].double()).to(s["x"].dtype).double()
        rms = ((h * h).sum(1) / h.shape[1] + s["eps"]) ** 0.5
        y = h * (s["weight"].double() / rms[:, None])
        scale = y.abs().max(1).values / 127.0
        q = torch.round((h * s["weight"].double()) / (h * s["weight"].double()).abs().max(1, keepdim=True).values * 127.0)
        return {"y": q * scale[:, None], "scale": scale, "h": h if s["residual"] is not None else None}
    if case["op"] == "product":
        a = s["q"].double() * s["q_scale"].double()[:, None]
        out = torch.empty(case["batch"], case["out_dim"], dtype=torch.float64, device="cuda")
        for at in range(0, case["out_dim"], 16384):
            b = s["w"][at:at + 16384].double() * s["w_scale"][at:at + 16384].double()[:, None]
            out[:, at:at + 16384] = torch.einsum("bk,nk->bn", a, b)
        return out
    # The scores of the beams that stay, from log-probabilities in 64 bits; the rest are whole numbers.
    batch, beams, vocab = case["batch"], case["beams"], case["vocab"]
    x = s["logits"].double()
    if case["window"] and case["penalty"] != 1.0:
        p = float(torch.tensor(case["penalty"]).double())
        for j in range(case["window"]):
            at = s["hist"][:, j:j + 1].long()
            v = x.gather(1, at)
            v = torch.where(s["count"][:, None] > j, torch.where(v > 0, v / p, v * p), v)
            x.scatter_(1, at, v)
    logp = torch.log_softmax(x, dim=1)
    del x
    n = min(beams, vocab)
    offer = logp.topk(n, dim=1).values + s["scores"].double()[:, None]
    live = s["finished"][:, None] == 0
    offer = torch.where(live, offer, torch.full_like(offer, -_INF))
    offer[:, :1] = torch.where(live, offer[:, :1], s["scores"].double()[:, None])
    size = (s["lengths"][:, None] + live.int()).double().pow(case["alpha"])
    ranked = (offer / size).view(batch, -1).topk(beams, dim=1).indices
    scores = offer.view(batch, -1).gather(1, ranked).reshape(-1)
    caches = None
    return {"tokens": None, "parents": None, "scores": scores, "lengths": None, "finished": None, "ring": None,
            "caches": caches}
