"""Measured cases of the grouped matrix products (forward, input gradient, weight gradient) and of the
orthogonalised update: their inputs, their plain form in elementary torch operations, the calls of the library, their
cost, and their values in 64 bits."""
import numpy as np
import torch

own = False

DTYPES = {"f64": torch.float64, "f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f64": 8, "f32": 4, "bf16": 2, "f16": 2}
COEF = (3.4445, -4.7750, 2.0315)   # the quintic of the orthogonalisation, the same in every step
EPS = 1e-7


def _g(name, op, dtype, groups, rows, n, k, idle=0, tail=0, out="same"):
    return {"name": name, "op": op, "dtype": dtype, "groups": groups, "rows": rows, "n": n, "k": k, "idle": idle,
            "tail": tail, "out": out}


def _o(name, dtype, batch, m, n, steps=5):
    return {"name": name, "op": "ortho", "dtype": dtype, "batch": batch, "m": m, "n": n, "steps": steps}


def listed():
    return [
        # serving: a handful of rows, each of another expert; latency and the read of the weights
        _g("forward, single rows", "forward", "bf16", 16, 8, 1024, 512, idle=8),
        # serving a batch of 64 requests with two experts a row: a few rows for each of 32 experts
        _g("forward, few rows", "forward", "bf16", 32, 128, 2816, 2048),
        # a training batch of ordinary size
        _g("forward, batch", "forward", "bf16", 16, 8192, 2816, 2048, tail=192),
        # the largest: long sequences through wide experts
        _g("forward, largest", "forward", "bf16", 8, 32768, 7168, 4096),
        # the benchmark's own dimensions (d = 50 inputs, m = 1024 features) in the type of the GP path
        _g("forward, d = 50 in 64 bits", "forward", "f64", 12, 65536, 1024, 50),
        # gradient of the inputs at odd sizes, one expert without rows
        _g("input gradient, odd", "dx", "f16", 7, 5003, 1111, 1403, idle=1, tail=5),
        # gradient of the inputs in single precision
        _g("input gradient, 32 bits", "dx", "f32", 8, 6144, 2048, 1408),
        # gradient of the weights of the batch above, accumulated in a 32-bit buffer as optimisers keep it
        _g("weight gradient, batch", "dw", "bf16", 16, 8192, 2816, 2048, tail=192, out="f32"),
        # Gram matrices of the rows of eight local experts (m = 1024), the type of the GP path
        _g("weight gradient, m = 1024 in 64 bits", "dw", "f64", 8, 65536, 1024, 1024),
        # the update of one small matrix: latency
        _o("orthogonalise, small", "f32", 1, 128, 50),
        # the updates of the weights of 16 experts at once
        _o("orthogonalise, experts", "bf16", 16, 1024, 2816),
        # the update of one large matrix
        _o("orthogonalise, largest", "f32", 1, 4096, 4096),
    ]


def _log(rng, lo, hi):
    return int(round(np.exp(rng.uniform(np.log(lo), np.log(hi)))))


def _extent(rng, lo, hi):
    """A size between lo and hi: any, a multiple of 8, or a multiple of 64."""
    v = _log(rng, lo, hi)
    step = rng.choice([1, 8, 64])
    return min(max(lo, v // step * step), hi)


def draw(rng):
    if rng.random() < 0.3:
        dtype = rng.choice(["f32", "bf16", "f16", "f64"])
        most = 4e10 if dtype == "f64" else 5e11
        while True:
            c = _o("", dtype, rng.choice([1, 1, 2, 4, 8, 24]), _extent(rng, 16, 4096), _extent(rng, 16, 4096), rng.choice([3, 5, 5, 6]))
            if work(c)["flops"] <= most:
                break
    else:
        dtype = rng.choice(["bf16", "bf16", "bf16", "f16", "f16", "f32", "f64"])
        most = {"f64": 1e11, "f32": 2e11}.get(dtype, 1e12)
        while True:
            op = rng.choice(["forward", "forward", "dx", "dw"])
            groups = _log(rng, 1, 64)
            out = "f32" if op == "dw" and dtype in ("bf16", "f16") and rng.random() < 0.5 else "same"
            c = _g("", op, dtype, groups, _log(rng, 1, 32768), _extent(rng, 16, 8192), _extent(rng, 16, 8192),
                   idle=rng.randrange(groups // 2 + 1) if rng.random() < 0.4 else 0, tail=rng.choice([0, 0, 1, 100]), out=out)
            w = work(c)
            if w["flops"] <= most and w["bytes"] <= 8e8 and groups * c["n"] * c["k"] <= 1 << 28:
                break
    del c["name"]
    return c


def _sizes(case, seed):
    """Rows of each group: random shares within a factor of three of one another, `idle` groups without rows."""
    rs = np.random.RandomState(seed % (1 << 31))
    groups, rows = case["groups"], case["rows"]
    share = rs.uniform(0.5, 1.5, groups)
    share[rs.permutation(groups)[:case["idle"]]] = 0.0
    ends = np.floor(np.cumsum(share) / share.sum() * rows + 0.5).astype(np.int64)
    ends[-1] = rows
    if share[-1] == 0.0:   # the last busy group takes the remainder, not an idle one behind it
        last = int(np.nonzero(share)[0][-1])
        ends[last:] = rows
    return np.diff(np.concatenate([[0], ends]))


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    rand_in = torch.float64 if case["dtype"] == "f64" else torch.float32

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device=dev, dtype=rand_in) * scale).to(dt)

    if case["op"] == "ortho":
        b, m, n = case["batch"], case["m"], case["n"]
        r = min(8, m, n)   # a gradient: a few strong directions over noise
        u = torch.randn(b, m, r, generator=gen, device=dev, dtype=rand_in)
        v = torch.randn(b, r, n, generator=gen, device=dev, dtype=rand_in)
        s = torch.logspace(0.0, -1.5, r, device=dev, dtype=rand_in)
        grad = 1e-3 * (torch.bmm(u * s, v) + torch.randn(b, m, n, generator=gen, device=dev, dtype=rand_in))
        return {"case": dict(case), "grad": grad.to(dt), "out": torch.empty(b, m, n, device=dev, dtype=dt)}
    groups, rows, n, k = case["groups"], case["rows"], case["n"], case["k"]
    sizes = _sizes(case, seed)
    ends = np.concatenate([[0], np.cumsum(sizes)])
    total = rows + case["tail"]
    st = {"case": dict(case), "longest": int(sizes.max()), "total": total,
          "offsets": torch.from_numpy(ends).to(dev)}
    if case["op"] == "dw":
        st["x"], st["dy"] = normal(total, k), normal(total, n)
        st["out"] = torch.empty(groups, n, k, device=dev, dtype=torch.float32 if case["out"] == "f32" else dt)
    else:
        # forward: weights n x k, k contiguous; input gradient of a layer k -> n: the same weights, summed over n
        st["x"] = normal(total, k if case["op"] == "forward" else n)
        st["w"] = normal(groups, n, k, scale=k ** -0.5)
        st["out"] = torch.zeros(total, n if case["op"] == "forward" else k, device=dev, dtype=dt)
    return st


def _padded(x, offsets, longest):
    """Rows of every group, padded with zeros to the longest one: (groups, longest, columns), and which are rows."""
    at = offsets[:-1, None] + torch.arange(longest, device=x.device)[None, :]
    real = at < offsets[1:, None]
    at = torch.clamp(at, max=x.shape[0] - 1)
    return torch.where(real[:, :, None], x[at], 0.0), at, real


def _plain_products(st):
    case = st["case"]
    wide = torch.float64 if case["dtype"] == "f64" else torch.float32
    x, at, real = _padded(st["x"].to(wide), st["offsets"], st["longest"])
    if case["op"] == "dw":
        dy = _padded(st["dy"].to(wide), st["offsets"], st["longest"])[0]
        return torch.bmm(dy.transpose(1, 2), x).to(st["out"].dtype)
    w = st["w"].to(wide)
    y = torch.bmm(x, w.transpose(1, 2) if case["op"] == "forward" else w)
    out = torch.zeros(st["total"], y.shape[2], device=y.device, dtype=st["out"].dtype)
    out[at[real]] = y[real].to(out.dtype)
    return out


def _plain_ortho(st):
    case = st["case"]
    a, b, c = COEF
    x = st["grad"].to(torch.float64 if case["dtype"] == "f64" else torch.float32)
    x = x / (x.square().sum((1, 2), keepdim=True).sqrt() + EPS)
    tall = case["m"] > case["n"]
    for _ in range(case["steps"]):
        p = torch.bmm(x.transpose(1, 2), x) if tall else torch.bmm(x, x.transpose(1, 2))
        q = b * p + c * torch.bmm(p, p)
        x = a * x + (torch.bmm(x, q) if tall else torch.bmm(q, x))
    return x.to(st["out"].dtype)


def run(st):
    case = st["case"]
    if own:
        from gp_amd import lib
        if case["op"] == "ortho":
            return lib.orthogonalize(st["grad"], st["out"], steps=case["steps"], eps=EPS)
        if case["op"] == "dw":
            return lib.grouped_gemm_dw(st["x"], st["dy"], st["offsets"], st["out"])
        return lib.grouped_gemm(st["x"], st["w"], st["offsets"], st["out"], w_kc=case["op"] == "forward")
    return _plain_ortho(st) if case["op"] == "ortho" else _plain_products(st)


def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "ortho":
        s, l = min(case["m"], case["n"]), max(case["m"], case["n"])
        # per step: half of X X^T and half of A A (both symmetric), and the product with X
        return {"bytes": 2 * e * case["batch"] * s * l, "flops": case["batch"] * case["steps"] * (3 * s * s * l + s ** 3)}
    busy = min(case["groups"] - case["idle"], case["rows"])
    rows, n, k = case["rows"], case["n"], case["k"]
    weights = (case["groups"] * n * k * (4 if case["out"] == "f32" else e)) if case["op"] == "dw" else busy * n * k * e
    return {"bytes": rows * (n + k) * e + weights + 8 * (case["groups"] + 1), "flops": 2 * rows * n * k}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "ortho":
        a, b, c = COEF
        done = []
        for g in st["grad"]:
            x = g.double()
            if x.shape[0] > x.shape[1]:
                x = x.T.contiguous()
            x = x / (torch.linalg.norm(x) + EPS)
            for _ in range(case["steps"]):
                p = x @ x.T
                px = p @ x
                x = a * x + b * px + c * (p @ px)
            done.append(x.T if case["m"] > case["n"] else x)
        return torch.stack(done)
    ends = st["offsets"].tolist()
    spans = list(zip(ends[:-1], ends[1:]))
    if case["op"] == "dw":
        return torch.stack([st["dy"][i:j].double().T.contiguous() @ st["x"][i:j].double() for i, j in spans])
    y = torch.zeros(st["total"], st["out"].shape[1], device=st["x"].device, dtype=torch.float64)
    for w, (i, j) in zip(st["w"], spans):
        if j > i:
            y[i:j] = st["x"][i:j].double() @ (w.double().T.contiguous() if case["op"] == "forward" else w.double())
    return y
