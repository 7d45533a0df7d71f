"""Plain forms of the beam search's operators, in 64 bits or whole numbers."""
import numpy as np


def beam_scores(logits, scores, done, done_token):
    """S (beams, vocab) of one request in f64, -inf where there is no candidate."""
    x = logits.astype(np.float64)
    out = np.full(x.shape, -np.inf)
    for b, s in enumerate(scores.astype(np.float64)):
        if not np.isfinite(s):
            continue
        if done is not None and done[b]:
            out[b, done_token if done_token < x.shape[1] else 0] = s
            continue
        if np.isnan(x[b]).any() or np.isposinf(x[b]).any() or np.isneginf(x[b]).all():
            continue
        top = x[b].max()
        lse = np.log(np.exp(x[b] - top).sum()) + top
        out[b] = s + x[b] - lse
    return out


def fork_ref(parent, kv_len, table, page, n_pages, pinned, ld_out):
    n = len(parent)
    out = np.full((n, ld_out), -1, np.int32)
    lens, opens = np.zeros(n, np.int32), [-1] * n
    full, first = set() if pinned is None else set(np.flatnonzero(pinned).tolist()), {}
    for i, p in enumerate(parent):
        if not 0 <= p < len(kv_len):
            continue
        lens[i] = max(int(kv_len[p]), 0)
        want = -(-int(lens[i]) // page)
        have = min(want, table.shape[1])
        for j in range(have):
            id_ = int(table[p, j])
            if not 0 <= id_ < n_pages:
                continue
            out[i, j] = id_
            if j == want - 1 and lens[i] % page:
                opens[i] = id_
                first.setdefault(id_, i)
            else:
                full.add(id_)
    held = full | set(first)
    free = [i for i in range(n_pages) if i not in held]
    src, dst, tok = (np.full(n, v, np.int32) for v in (-1, -1, 0))
    wants = 0
    for i in range(n):
        id_ = opens[i]
        if id_ < 0 or (id_ not in full and first[id_] == i):
            continue
        new = free[wants] if wants < len(free) else -1
        wants += 1
        out[i, -(-int(lens[i]) // page) - 1] = new
        src[i], dst[i], tok[i] = id_, new, lens[i] % page
    left = free[wants:]
    rest = np.full(n_pages, -1, np.int32)
    rest[:len(left)] = left
    return out, lens, src, dst, tok, rest, np.array([len(left), wants], np.int64)


def compact_ref(kv_len, table, page, n_pages, ld_out):
    rows = []
    for n, row in zip(kv_len, table):
        have = min(-(-max(int(n), 0) // page), table.shape[1])
        rows.append([int(i) if 0 <= i < n_pages else -1 for i in row[:have]])
    held = sorted({i for r in rows for i in r if i >= 0})
    n = len(held)
    holes = sorted(set(range(n)) - set(held))
    moves = [i for i in held if i >= n]
    to = {**{i: i for i in held}, **dict(zip(moves, holes)), -1: -1}
    out = np.full((len(rows), ld_out), -1, np.int32)
    for s, r in enumerate(rows):
        out[s, :len(r)] = [to[i] for i in r]
    src, dst = (np.full(n_pages // 2, -1, np.int32) for _ in range(2))
    src[:len(moves)], dst[:len(moves)] = moves, holes
    return out, src, dst, np.array([n, len(moves)], np.int64)
