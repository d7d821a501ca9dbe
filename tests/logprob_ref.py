"""Log probabilities, ranks, entropies and best ids of one row of logits in 64
bits, and how far a computation in the operator's own arithmetic may be off."""
import numpy as np

EPS = 2.0 ** -24


def best_ids(x, k):
    """The first k ids: larger logits first, of equal ones the lower id; no NaN, no -inf."""
    some = np.flatnonzero(x > -np.inf)
    return some[np.argsort(-x[some], kind="stable")][:k]


def row(x, token, k, temperature=1.0):
    """x in 64 bits. {name: value}, with "_tol" entries; probabilities None for a
    row without a distribution."""
    x = np.asarray(x, np.float64)
    v = len(x)
    inside = 0 <= token < v
    xt = x[token] if inside else -np.inf
    rank = 0 if not inside or np.isnan(xt) else 1 + int((x > xt).sum()) + int((x[:token] == xt).sum())
    ids = best_ids(x, k)
    out = {"rank": rank, "ids": np.concatenate([ids, np.full(k - len(ids), -1)]).astype(np.int32)}
    greedy = not temperature > 0
    m = np.max(x[~np.isnan(x)], initial=-np.inf)
    if m == -np.inf or (not greedy and (np.isnan(x).any() or m == np.inf)):
        return {**out, "lp": None, "h": None, "best": None}
    if greedy:
        lp = np.full(v, -np.inf)
        lp[np.flatnonzero(x == m)[0]] = 0.0
        return {**out, "lp": lp[token] if inside else -np.inf, "h": 0.0, "lp_tol": 0.0, "h_tol": 0.0,
                "best": np.concatenate([lp[ids], np.full(k - len(ids), -np.inf)]), "best_tol": np.zeros(k)}
    t = np.where(x == -np.inf, -np.inf, 0.0) if np.isinf(temperature) else (x - m) / float(np.float32(temperature))
    e = np.exp(t)
    tops = int((x == m).sum())
    rest = e[x != m].sum()
    z = tops + rest
    log_z = np.log1p(tops - 1 + rest)
    p = e / z
    some = p > 0
    h = log_z - (p[some] * t[some]).sum()
    # Terms: the hardware's exponential 2 eps; its argument (base 2) has three
    # roundings, 3 eps |t|, and so has the term, relatively. Sums: 16 additions in a
    # lane, 7 over lanes; or 10 and 6 with the maximum's own term among them, where the
    # sum is at least 3, 3/2 times as much of what is left without it. log Z of
    # 1 + (Z - 1) errs by the error of Z - 1 over Z.
    # The entropy's other part sums e t alike, with one product's rounding more.
    # Results are rounded to fp32; the given logit's own t has the rate's rounding
    # (fp64 else).
    share = (z - 1) / z
    a1, a2 = -(p[some] * t[some]).sum(), (p[some] * t[some] ** 2).sum()
    z_tol = EPS * (27 * share + 3 * a1)
    h_tol = z_tol * (1 + a1) + EPS * (30 * a1 + 3 * a2 + h)
    lp = t - log_z
    lp = np.where(lp < -3.4028236e38, -np.inf, lp)  # what fp32 rounds it to

    def tol(ids):
        tt = np.abs(np.where(np.isfinite(t[ids]), t[ids], 0.0))
        return z_tol + EPS * (tt + np.where(np.isfinite(lp[ids]), np.abs(lp[ids]), 0.0)) * 1.01
    return {**out, "lp": lp[token] if inside else -np.inf, "lp_tol": float(tol([token])[0]) if inside else 0.0, "h": h,
            "h_tol": h_tol, "best": np.concatenate([lp[ids], np.full(k - len(ids), -np.inf)]),
            "best_tol": np.concatenate([tol(ids), np.zeros(k - len(ids))])}
