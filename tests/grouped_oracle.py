"""Plain 64-bit forms of the grouped products and of the orthogonalised update (CPU or GPU torch tensors), and the
tolerances that follow from the formulas."""
import numpy as np
import torch

#: half a step of each type, relative to the value
HALF = {torch.float64: 2.0 ** -53, torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
#: smallest step of each type (results below the normal range are off by half of it)
TINY = {torch.float64: 2.0 ** -1074, torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}
COEF = (3.4445, -4.7750, 2.0315)


def spans(offsets, rows):
    """Rows of every group as the interface reads the table: ends clamped to [0, rows], a decreasing pair is empty."""
    o = [min(max(int(v), 0), rows) for v in offsets]
    return [(a, max(a, b)) for a, b in zip(o[:-1], o[1:])]


def grouped(x, w, offsets, out, w_kc=True, alpha=1.0, beta=0.0):
    """(result, bound of its error)."""
    x64, w64, old = x.double(), w.double(), out.double()
    y, tol = old.clone(), torch.zeros_like(old)
    k = x.shape[1]
    unit = 2.0 ** -52 if x.dtype == torch.float64 else 2.0 ** -23   # an addition inside the matrix instruction, either way
    for g, (a, b) in enumerate(spans(offsets, x.shape[0])):
        if b > a:
            wg = (w64[g].T if w_kc else w64[g]).contiguous()
            y[a:b] = alpha * (x64[a:b] @ wg) + (beta * old[a:b] if beta else 0.0)
            size = abs(alpha) * (x64[a:b].abs() @ wg.abs()) + (abs(beta) * old[a:b].abs() if beta else 0.0)
            tol[a:b] = (k + 3) * unit * size + HALF[out.dtype] * y[a:b].abs() + TINY[out.dtype]
    return y, tol


def grouped_dw(x, dy, offsets, out, alpha=1.0, beta=0.0):
    x64, z64, old = x.double(), dy.double(), out.double()
    c, tol = torch.empty_like(old), torch.empty_like(old)
    unit = 2.0 ** -52 if x.dtype == torch.float64 else 2.0 ** -23
    for g, (a, b) in enumerate(spans(offsets, x.shape[0])):
        zt = z64[a:b].T.contiguous()
        c[g] = alpha * (zt @ x64[a:b]) + (beta * old[g] if beta else 0.0)
        size = abs(alpha) * (zt.abs() @ x64[a:b].abs()) + (abs(beta) * old[g].abs() if beta else 0.0)
        tol[g] = (b - a + 3) * unit * size + HALF[out.dtype] * c[g].abs() + TINY[out.dtype]
    return c, tol


def orthogonalize(g, steps=5, coef=None, eps=1e-7):
    """(result, bound of the relative error of one matrix in the Frobenius norm).

    An error e of X_k reaches the result multiplied by at most prod_{j >= k} L_j, L_j = max |p_j'| over the singular values
    that step j can meet (the derivative of an odd matrix function acts through divided differences of p_j, which the mean
    value theorem bounds).  A step makes an error of at most u (4 + sqrt(2 side)) sum|terms| (random signs in its dot
    products), u: 2^-22 for operands held to 22 bits or more, 2^-52 in double."""
    triples = [COEF] * steps if coef is None else ([tuple(coef)] * steps if np.ndim(coef) == 1 else [tuple(c) for c in coef])
    x = g.double()
    x = x / (torch.linalg.norm(x) + eps)
    u = 2.0 ** -52 if g.dtype == torch.float64 else 2.0 ** -22
    made, grow, top = [u * float(torch.linalg.norm(x))], [], 1.0
    for a, b, c in triples:
        p = x @ x.T
        px = p @ x
        ppx = p @ px
        terms = sum(abs(k) * float(torch.linalg.norm(t)) for k, t in ((a, x), (b, px), (c, ppx)))
        made.append(u * (4 + (2.0 * max(g.shape)) ** 0.5) * terms)
        s = np.linspace(0.0, top, 4001)
        grow.append(max(1.0, float(np.max(np.abs(a + 3 * b * s ** 2 + 5 * c * s ** 4)))))
        top = float(np.max(np.abs(a * s + b * s ** 3 + c * s ** 5))) * 1.0001
        x = a * x + b * px + c * ppx
    err = 0.0
    for k, e in enumerate(made):
        err += e * float(np.prod(grow[k:])) if k < len(grow) else e
    norm = float(torch.linalg.norm(x))
    return x, (err / norm if norm else 0.0) + HALF[g.dtype]
