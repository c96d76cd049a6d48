"""Drawing and verifying tokens by the definition, in float64 on the host."""
import numpy as np
import torch


def distribution(row, temperature=1.0, top_k=0, top_p=1.0):
    """Weights of one row's tokens over their sum (zeros for a row without a token)."""
    l = torch.as_tensor(row).double().cpu().numpy().copy()
    l[np.isnan(l)] = -np.inf
    top = l.max()
    if top == -np.inf:
        return np.zeros(l.size)
    if not temperature > 0:
        w = np.zeros(l.size)
        w[int(np.argmax(l))] = 1.0
        return w
    with np.errstate(invalid="ignore"):
        w = (l == np.inf).astype(np.float64) if top == np.inf else np.where(l > -np.inf, np.exp((l - top) / temperature), 0.0)
    order = np.argsort(-l, kind="stable")
    if top_k > 0:
        w[order[top_k:]] = 0.0
    if top_p < 1:
        run = np.cumsum(w[order])
        n = max(1, int(np.searchsorted(run, max(top_p, 0.0) * run[-1], side="left")) + 1)
        w[order[n:]] = 0.0
    return w / w.sum()


def pick(p, u):
    """The lowest index whose running sum passes u of the whole, -1 without mass."""
    run = np.cumsum(p)
    if not run[-1] > 0:
        return -1
    u = 0.0 if np.isnan(u) else min(max(u, 0.0), 1.0)
    at = int(np.searchsorted(run, u * run[-1], side="right"))
    return at if at < p.size else int(np.flatnonzero(p)[-1])


def per(value, n, default):
    """n numbers of a parameter given as None, a number (taken as float32) or a tensor."""
    if value is None:
        return [default] * n
    if isinstance(value, torch.Tensor):
        return value.double().cpu().tolist()
    return [float(np.float32(value))] * n


def sample(logits, uniforms, temperature=None, top_k=None, top_p=None):
    """(tokens, distributions)."""
    N = logits.shape[0]
    t, k, p = per(temperature, N, 1.0), per(top_k, N, 0), per(top_p, N, 1.0)
    rows = [distribution(logits[n], t[n], int(k[n]), p[n]) for n in range(N)]
    u = uniforms.double().cpu().tolist()
    return torch.tensor([pick(r, x) for r, x in zip(rows, u)], dtype=torch.int64), rows


def verify(logits, drafts, accept, draw, draft_probs=None, cu=None, temperature=None, top_k=None, top_p=None):
    """(tokens, accepted) of verify_drafts."""
    B, K = drafts.shape
    V = logits.shape[-1]
    flat = logits.reshape(-1, V).cpu()
    cu = [b * (K + 1) for b in range(B + 1)] if cu is None else [min(max(int(c), 0), flat.shape[0]) for c in cu]
    t, k, p = per(temperature, B, 1.0), per(top_k, B, 0), per(top_p, B, 1.0)
    tokens = torch.full((B, K + 1), -1, dtype=torch.int64)
    accepted = torch.zeros(B, dtype=torch.int32)
    x, a, u = drafts.cpu(), accept.double().cpu(), draw.double().cpu()
    for b in range(B):
        rows = min(max(cu[b + 1] - cu[b], 0), K + 1)
        for i in range(rows):
            dist = distribution(flat[cu[b] + i], t[b], int(k[b]), p[b])
            if i == rows - 1:
                tokens[b, i] = pick(dist, float(u[b]))
                break
            d = int(x[b, i])
            known = 0 <= d < V
            if known:
                q = np.zeros(V)
                if draft_probs is None:
                    q[d] = 1.0
                else:
                    q = np.maximum(draft_probs[b, i].double().cpu().numpy(), 0.0)
                if float(a[b, i]) * q[d] < dist[d]:
                    tokens[b, i] = d
                    accepted[b] += 1
                    continue
                with np.errstate(invalid="ignore"):
                    rest = dist - q
                rest = np.where(rest > 0, rest, 0.0)
                if draft_probs is None:
                    rest = dist.copy()
                    rest[d] = 0.0
                if rest.sum() > 0:
                    dist = rest
            tokens[b, i] = pick(dist, float(u[b]))
            break
    return tokens, accepted
