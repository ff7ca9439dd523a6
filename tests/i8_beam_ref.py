"""Plain 64-bit restatements of the 8-bit norm, the 8-bit unembedding product and the beam
step, for the tests of the kernels. numpy only."""
import numpy as np


def norm_i8(h, weight, eps):
    """h: the rows after the residual's addition, rounded to their type, as float64.
    Returns (q int8, scale float64); a row with a NaN or infinity has scale NaN and q 0."""
    h, w = np.asarray(h, np.float64), np.asarray(weight, np.float64)
    with np.errstate(all="ignore"):
        t = h * w
        bad = ~(np.isfinite(t).all(1) & np.isfinite(h).all(1))
        top = np.abs(t).max(1, keepdims=True)
        q = np.where((top > 0) & ~bad[:, None], np.rint(t * 127.0 / np.where(top > 0, top, 1.0)), 0.0)
        q = np.nan_to_num(q)
        scale = top[:, 0] / 127.0 / np.sqrt((h * h).mean(1) + np.float64(np.float32(eps)))
    scale[bad] = np.nan
    return q.astype(np.int8), scale


def product_i8(q, scale, wq, ws):
    acc = q.astype(np.float64) @ wq.astype(np.float64).T  # whole numbers below 2^53: exact
    return acc * np.asarray(scale, np.float64)[:, None] * np.asarray(ws, np.float64)[None, :]


def penalise(x, ring, penalty):
    """One row (float32): per ring slot in order x / p or x * p in fp32 (Sampler.pas:285-303)."""
    x = x.copy()
    p = np.float32(penalty)
    with np.errstate(all="ignore"):
        for t in ring:
            if 0 <= t < len(x):
                x[t] = x[t] / p if x[t] > 0 else x[t] * p
    return x


def beam_step(logits, batch, beams, state, stop_ids=(), pad=0, penalty=1.0, alpha=0.0):
    """logits float32 [rows, vocab]; state: dict of scores f32, lengths, finished, and hist, pos,
    count where there are rings. Returns (tokens, parents, new state, ranks, offers): ranks is
    the float64 rank of every pick (-inf: none), offers[prompt] maps (beam, token) to its rank."""
    rows, vocab = logits.shape
    out = {k: np.array(v, copy=True) for k, v in state.items()}
    tokens, parents = np.zeros((batch, beams), np.int32), np.zeros((batch, beams), np.int32)
    ranks, offers = np.full((batch, beams), -np.inf), []
    window = state["hist"].shape[1] if "hist" in state else 0
    for g in range(batch):
        cand = []
        for b in range(beams):
            r = g * beams + b
            score, length, done = np.float64(state["scores"][r]), int(state["lengths"][r]), state["finished"][r] != 0
            if done:
                if score > -np.inf:
                    cand.append((score / float(max(length, 1)) ** alpha, b, 0, pad, score, length))
                continue
            if not score > -np.inf:
                continue
            x = logits[r]
            if window and penalty != 1.0:
                x = penalise(x, state["hist"][r][:min(max(int(state["count"][r]), 0), window)], penalty)
            x = x.astype(np.float64)
            if np.isnan(x).any() or x.max() == np.inf or x.max() == -np.inf:
                continue
            top = x.max()
            lse = top + np.log(np.exp(x - top).sum())
            order = np.argsort(-x, kind="stable")[:beams]
            for i, v in enumerate(order):
                s = score + (x[v] - lse)
                if s > -np.inf:
                    cand.append((s / float(max(length + 1, 1)) ** alpha, b, i, int(v), s, length + 1))
        offers.append({(c[1], c[3]): c[0] for c in cand})
        cand.sort(key=lambda c: (-c[0], c[1], c[2]))
        for k in range(beams):
            r = g * beams + k
            if k >= len(cand):
                tokens[g, k], parents[g, k] = pad, k
                out["scores"][r], out["finished"][r] = -np.inf, 0
                out["lengths"][r] = state["lengths"][r]
                src, fresh = r, False
            else:
                rank, b, _, tok, s, length = cand[k]
                src = g * beams + b
                fresh = state["finished"][src] == 0
                tokens[g, k], parents[g, k], ranks[g, k] = tok, b, rank
                out["scores"][r], out["lengths"][r] = np.float32(s), length
                out["finished"][r] = int(tok in stop_ids) if fresh else 1
            if window:
                out["hist"][r] = state["hist"][src]
                at, held = int(state["pos"][src]) % window, int(state["count"][src])
                if fresh:
                    out["hist"][r][at] = tokens[g, k]
                    at, held = (at + 1) % window, held + 1 if held < window else held
                out["pos"][r], out["count"][r] = at, held
    return tokens, parents, out, ranks, offers
