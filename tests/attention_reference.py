"""Attention and its gradients from the definition in 64 bits, and how far the kernels' results may be from them.

With u = 2^-24, h half a step of the type, A = |q||k|^T scale: a score is a 32-bit sum of D exact products, off by (D + 4) u A with its exponent's rounding; e is the largest of a row, so that a probability is off by
2 e relative and, rounded, by h. o is sum p v / sum p over rounded p, off by (2 h + 4 e) sum p|v| and its rounding. lse is that of the rounded sum, off by h, and probabilities backward by as much: dv (2 h + 4 e) sum p|dO|. dO v is off by (D + 1) u |dO||v|, the sum dO o by what o before its rounding is (with 2 h^2 |o| from
that of what it left), and by (D + 1) u |dO||o|:
dS by p times these and (2 h + 4 e)|dS|; dk by the sums of these with |q|, dq with |k| + |c|: it is sum dS k - (sum dS) c, the
second 0 but for these errors, with c a mean of the first 64 keys, as large as their largest at most. 32-bit sums over n rows or keys add n u of the sum of magnitudes. A value below the type's smallest normal one is off by half of its smallest step:
float16's is 2^-25 of a row's largest probability forward, which is at most the row's sum (o: 2^-25 sum |v|); backward probabilities are held times 2^14 (dv: 2^-39 sum |dO|) and dS times the power of two 2^e that keeps
B = 2 D max|dO| max|v| within 2^15: 2^e > 2^14 / B, half a step 2^-25 / 2^e < B 2^-39 (dq: scale B 2^-39 sum |k| over the keys it sees, dk alike with |q|). bfloat16 has float32's range."""
import torch

U = 2.0 ** -24


def visible(n, m, causal):
    seen = torch.ones(n, m, dtype=torch.bool, device="cuda")
    return seen.tril(m - n) if causal else seen


def reference(q, k, v, do, spans, causal=True, scale=None):
    """q [N, Hq, D], k, v [M, Hk, D] (any type), spans (q0, q1, k0, k1) of each sequence: {name: (values, tolerance)}"""
    h = 0.5 * torch.finfo(q.dtype).eps
    small = torch.finfo(q.dtype).smallest_normal * h * 2
    q, k, v = (t.detach().double() for t in (q, k, v))
    do = None if do is None else do.double()
    N, Hq, D = q.shape
    Hk, G = k.shape[1], Hq // k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    narrow = q.shape[0] and k.shape[0] and h == 2.0 ** -11
    lost = 2 * D * float(do.abs().max()) * float(v.abs().max()) * 2.0 ** -39 if narrow and do is not None else 0.0
    out = {n: (torch.zeros_like(t), torch.zeros_like(t)) for n, t in (("o", q), ("dq", q), ("dk", k), ("dv", k))}
    for q0, q1, k0, k1 in spans:
        n, m = q1 - q0, k1 - k0
        if not n or not m:
            continue
        seen = visible(n, m, causal)
        for head in range(Hq):
            e = head // G
            a, b, c = q[q0:q1, head], k[k0:k1, e], v[k0:k1, e]
            err = ((D + 4) * U * scale * (a.abs() @ b.abs().T)).masked_fill(~seen, 0).amax(1, keepdim=True)
            p = torch.nan_to_num(torch.softmax((scale * a @ b.T).masked_fill(~seen, float("-inf")), 1), nan=0.0)
            o = p @ c
            out["o"][0][q0:q1, head] = o
            out["o"][1][q0:q1, head] = (2 * h + 4 * err + (m + 8) * U) * (p @ c.abs()) + (2.0 ** -25 * (seen.double() @ c.abs()) if narrow else 0)
            if do is None:
                continue
            g = do[q0:q1, head]
            dp = g @ c.T
            delta = (g * o).sum(1, keepdim=True)
            ds = p * (dp - delta)
            e_dp = (D + 1) * U * (g.abs() @ c.abs().T) + (2 * h * h + (D + 1) * U) * (g.abs() * o.abs()).sum(1, keepdim=True) + 1.1 * (g.abs() * out["o"][1][q0:q1, head]).sum(1, keepdim=True)
            e_ds = p * e_dp + (2 * h + 4 * err + 4 * U) * ds.abs()
            e_ds = e_ds + lost * seen
            out["dv"][0][k0:k1, e] += p.T @ g
            out["dv"][1][k0:k1, e] += (p * (2 * h + 4 * err + (n * G + 8) * U)).T @ g.abs() + (2.0 ** -39 * (seen.double().T @ g.abs()) if narrow else 0)
            out["dq"][0][q0:q1, head] = scale * ds @ b
            c = b[:64].abs().amax(0)
            out["dq"][1][q0:q1, head] = scale * (e_ds + m * U * ds.abs()) @ (b.abs() + c)
            out["dk"][0][k0:k1, e] += scale * ds.T @ a
            out["dk"][1][k0:k1, e] += scale * (e_ds + n * G * U * ds.abs()).T @ a.abs()
    return {name: (want, 1.01 * (tol + h * want.abs() + small)) for name, (want, tol) in out.items()}


def check(got, want, tol, what=""):
    off = (got.detach().double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} values, first {bad.nonzero()[0].tolist()}, off by up to {float((off / tol).nan_to_num(nan=1e9).max()):.3g} tolerances"
