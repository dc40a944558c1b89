"""The operators at the head of a network in 64 bits, from their definitions (numpy)."""
import numpy as np

U = 2.0 ** -24          # half a step of float32, relative


def layer_norm(x, gamma, beta, eps):
    x = np.asarray(x, np.float64)
    mean = x.mean(0)
    rstd = 1.0 / np.sqrt(((x - mean) ** 2).mean(0) + eps)
    return (x - mean) * rstd * gamma.astype(np.float64)[:, None] + beta.astype(np.float64)[:, None], mean, rstd


def layer_norm_backward(x, dy, gamma, mean, rstd):
    """mean, rstd: the float32 values that the kernel is given"""
    x, dy, mean, rstd = (np.asarray(a, np.float64) for a in (x, dy, mean, rstd))
    xh = (x - mean) * rstd
    g = dy * gamma.astype(np.float64)[:, None]
    return rstd * (g - g.mean(0) - xh * (g * xh).mean(0)), (dy * xh).sum(1), dy.sum(1)


def keys(y):
    """[channels, columns] -> what sorts ascending into the operator's order: not-a-number first, then descending"""
    y = np.asarray(y, np.float64)
    return np.where(np.isnan(y), -np.inf, -np.where(np.isnan(y), 0.0, y)), ~np.isnan(y)


def top_logits(y, k):
    """y [channels, columns] -> (channel, value) [k, columns]"""
    key, number = keys(y)
    channel = np.broadcast_to(np.arange(y.shape[0])[:, None], y.shape)
    order = np.lexsort((channel, key, number), axis=0)[:k]
    return order.astype(np.int32), np.take_along_axis(y, order, 0)


def distillation(y, index, z, w, t, weight_sum):
    """y [channels, columns], index and z [k, columns], w [columns] -> (dy, loss)"""
    y, z, w = (np.asarray(a, np.float64) for a in (y, z, w))
    c, n = y.shape
    dy, loss = np.zeros((c, n)), np.zeros(n)
    with np.errstate(all="ignore"):
        for f in range(n):
            ok = (index[:, f] >= 0) & (index[:, f] < c)
            zs, at = z[ok, f] / t, index[ok, f]
            if w[f] == 0 or not len(zs) or np.all(zs == -np.inf):
                continue
            a = y[:, f] / t
            log_p = a - a.max() - np.log(np.exp(a - a.max()).sum())
            top = zs[~np.isnan(zs)].max(initial=-np.inf)
            e = np.exp(np.where(zs == top, 0.0, zs - top))
            q = e / e.sum()
            live = ~(q == 0)
            loss[f] = w[f] * t * t * (q[live] * (np.log(q[live]) - log_p[at[live]])).sum()
            dense = np.zeros(c)
            np.add.at(dense, at, q)
            dy[:, f] = w[f] * t / weight_sum * (np.exp(log_p) - dense)
    return dy, loss


def sampling(y, u, t, k, top_p, min_p):
    """-> (category, share) [columns]"""
    channel, value = top_logits(y, k)
    value = value.astype(np.float64)
    n = y.shape[1]
    category, share = np.full(n, -1, np.int32), np.zeros(n)
    t, top_p, min_p = (float(np.float32(a)) for a in (t, top_p, min_p))
    for f in range(n):
        z = value[:, f]
        if not z[0] > -np.inf:
            continue
        with np.errstate(all="ignore"):
            e = np.exp(np.where(z == z[0], 0.0, (z - z[0]) / t))
        up_to = np.cumsum(e)
        kept = 1
        while kept < k and e[kept] > 0 and e[kept] >= min_p and (top_p >= 1 or up_to[kept - 1] < top_p * up_to[-1]):
            kept += 1
        total = up_to[kept - 1]
        drawn = min(int((up_to[:kept] <= float(u[f]) * total).sum()), kept - 1)
        category[f], share[f] = channel[drawn, f], e[drawn] / total
    return category, share
