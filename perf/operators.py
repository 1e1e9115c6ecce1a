"""What is measured of the adapter and list operators: their cases, their plain forms in elementary
torch operations, and the calls that a program makes of the library.

  lora_fwd  low-rank adapters of many requests beside a shared Linear projection:
            t[m] = A[e_m] x[m],  y[m] = act(W x[m] + bias + s[e_m] B[e_m] t[m]),  e_m = -1: no adapter
  lora_bwd  its gradients: g = dy act'(y), dt[m] = s[e_m] B[e_m]^T g[m], dx = g W + A[e_m]^T dt[m],
            dA[e] = sum over its rows of dt x^T, dB[e] = s[e] sum over its rows of g t^T
  clip      the global norm over a list of gradient tensors, and the clipping of all of them by it
  adam      one optimizer step over lists of tensors, with the gradients clipped by their global norm

`beside` is true where the projection's own product was made by another call: the adapters' part is then
added to what y (or dx) holds, which is how a program adds adapters to a product it already has.
"""
import torch

own = False

BETA1, BETA2, LR, EPS, CLIP_EPS = 0.9, 0.999, 1e-3, 1e-8, 1e-6

# The networks whose tensors the list cases take: the control network of the one-launch training step, and the MLP of
# the data-parallel training step.
SMALL_NET = "8-64-64-2"
LARGE_NET = "784-4096-4096-4096-10"


def listed():
    return [
        # one request of a served model: latency, the stream of W
        dict(name="fwd one token", op="lora_fwd", rows=1, n=4096, k=4096, rank=16, adapters=8, mix="shuffled", beside=False, act="none"),
        # a decode batch: every row has its own adapter, some have none
        dict(name="fwd 16 requests", op="lora_fwd", rows=16, n=4096, k=4096, rank=16, adapters=64, mix="shuffled", beside=False, act="none"),
        # a ragged evaluation batch through an odd-sized layer with its activation
        dict(name="fwd odd sizes", op="lora_fwd", rows=333, n=517, k=1000, rank=6, adapters=5, mix="shuffled", beside=False, act="relu"),
        # prompts of several requests, row after row, beside a projection that is already there
        dict(name="fwd prompts", op="lora_fwd", rows=8192, n=4096, k=4096, rank=16, adapters=8, mix="segments", beside=True, act="none"),
        # fine-tuning a small layer: latency
        dict(name="bwd small layer", op="lora_bwd", rows=64, n=64, k=128, rank=4, adapters=1, mix="one", beside=False, act="relu"),
        # fine-tuning one adapter on a full batch
        dict(name="bwd full batch", op="lora_bwd", rows=8192, n=4096, k=4096, rank=16, adapters=1, mix="one", beside=True, act="none"),
        # many adapters trained at once on one rank's rows of the MLP's first layer
        dict(name="bwd mixed adapters", op="lora_bwd", rows=1024, n=4096, k=784, rank=32, adapters=12, mix="shuffled", beside=False, act="relu"),
        # gradients of the control network: six small tensors, latency
        dict(name="clip control net", op="clip", shapes=SMALL_NET, copies=1, rank=0, pad=4),
        # gradients of rank-16 adapters of 128 square layers
        dict(name="clip adapters", op="clip", shapes="1024-1024", copies=128, rank=16, pad=4),
        # gradients of the MLP
        dict(name="clip mlp", op="clip", shapes=LARGE_NET, copies=1, rank=0, pad=4),
        # the same networks' optimizer steps
        dict(name="adam control net", op="adam", shapes=SMALL_NET, copies=1, rank=0, pad=4),
        dict(name="adam mlp", op="adam", shapes=LARGE_NET, copies=1, rank=0, pad=4),
    ]


def _log(rng, lo, hi):
    v = lo * (hi / lo) ** rng.random()
    return max(lo, min(hi, int(round(v))))


def _width(rng, lo, hi):
    v = _log(rng, lo, hi)
    r = rng.random()
    return v if r < 0.4 else max(4, v // 4 * 4) if r < 0.7 else max(lo, min(hi, 1 << (v.bit_length() - 1)))


def draw(rng):
    op = rng.choice(["lora_fwd", "lora_fwd", "lora_bwd", "lora_bwd", "clip", "adam"])
    if op.startswith("lora"):
        c = dict(op=op, rows=_log(rng, 1, 8192), n=_width(rng, 32, 4096), k=_width(rng, 32, 4096), rank=rng.choice([1, 2, 4, 5, 8, 12, 16, 24, 32, 48, 64]),
                 adapters=_log(rng, 1, 64), mix=rng.choice(["one", "segments", "shuffled"]), beside=rng.random() < 0.5, act=rng.choice(["none", "none", "relu", "tanh"]))
        if c["rows"] * c["n"] * c["k"] > 3_000_000_000:
            c["beside"] = True
        if c["rows"] * c["rank"] * (c["n"] + c["k"]) > 8192 * 16 * 8192:
            c["rank"] = max(1, 8192 * 16 * 8192 // (c["rows"] * (c["n"] + c["k"])))
        return c
    # hidden widths of one network, or adapters of many layers; `pad` 1 packs the tensors without alignment
    if rng.random() < 0.5:
        widths = [_width(rng, 4, 4096) for _ in range(rng.randint(2, 4))]
        if sum(u * v for u, v in zip(widths, widths[1:])) > 36_000_000:
            widths = [-(-v // 2) for v in widths]
        return dict(op=op, shapes="-".join(map(str, widths)), copies=1, rank=0, pad=rng.choice([4, 4, 1]))
    w = [_width(rng, 16, 2048) for _ in range(2)]
    return dict(op=op, shapes="-".join(map(str, w)), copies=_log(rng, 2, 128), rank=rng.choice([4, 8, 16, 32]), pad=rng.choice([4, 4, 1]))


def _sizes(case):
    """Elements of each tensor of a list case: weights and biases of a network, or both factors of every layer's adapter."""
    d = [int(v) for v in case["shapes"].split("-")]
    one = [n for i in range(len(d) - 1) for n in ([case["rank"] * d[i], d[i + 1] * case["rank"]] if case["rank"] else [d[i] * d[i + 1], d[i + 1]])]
    return one * case["copies"]


def _spans(case):
    """(offset, size) of each tensor in one flat buffer, and the buffer's length."""
    at, spans = 0, []
    for n in _sizes(case):
        spans.append((at, n))
        at += -(-n // case["pad"]) * case["pad"]
    return spans, at


def _row_adapters(case, gen, dev):
    m, e = case["rows"], case["adapters"]
    if case["mix"] == "one":
        return None
    if case["mix"] == "shuffled":  # one in sixteen rows without an adapter, as far as there are that many
        i = torch.randint(0, e, (m,), generator=gen, device=dev)
        off = torch.rand((m,), generator=gen, device=dev) < 1 / 16
        off[0] = False
        return torch.where(off, -1, i).to(torch.int32)
    # prompts of ragged lengths one after the other: each takes up to an eighth of the rows
    cut = torch.rand((16,), generator=gen, device=dev) + 0.2
    ends = (torch.cumsum(cut, 0) / cut.sum() * m).long()
    which = torch.randint(-1, e, (17,), generator=gen, device=dev)
    return which[torch.searchsorted(ends, torch.arange(m, device=dev), right=True).clamp(max=15)].to(torch.int32)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=dev)

    def uniform(bound, *shape):
        return (torch.rand(shape, generator=gen, device=dev) * 2 - 1) * bound

    s = {"case": case}
    if case["op"].startswith("lora"):
        m, n, k, r, e = (case[v] for v in ("rows", "n", "k", "rank", "adapters"))
        s["x"] = normal(m, k)
        s["w"] = None if case["beside"] else uniform(k ** -0.5, n, k)
        s["bias"] = None if case["beside"] else uniform(k ** -0.5, n)
        s["a"] = uniform(k ** -0.5, e, r, k)
        s["b"] = normal(e, n, r) * r ** -0.5
        s["scale"] = torch.rand((e,), generator=gen, device=dev) * 1.5 + 0.5
        s["idx"] = _row_adapters(case, gen, dev)
        s["t"] = torch.empty((m, r), device=dev)
        if case["op"] == "lora_fwd":
            s["y"] = normal(m, n)                   # beside: the projection's output; otherwise written
        else:
            s["t"] = _down(s["x"], s["a"], s["idx"])    # kept from the forward pass
            s["y"] = {"none": lambda v: v, "relu": torch.relu, "tanh": torch.tanh}[case["act"]](normal(m, n))
            s["dy"] = normal(m, n)
            s["dx"] = normal(m, k)                  # beside: the projection's part of the gradient
            s["da"], s["db"] = torch.empty_like(s["a"]), torch.empty_like(s["b"])
    else:
        spans, total = _spans(case)
        s["spans"] = spans
        s["g"] = normal(total) * 0.02
        # clipping binds: the norm is about 0.02 * sqrt(elements)
        s["max_norm"] = 0.01 * sum(v for _, v in spans) ** 0.5
        s["norm"], s["coef"] = torch.zeros(1, device=dev), torch.zeros(1, device=dev)
        if case["op"] == "adam":
            s["p"], s["m"] = uniform(0.05, total), normal(total) * 0.01
            s["v"] = s["m"].square() + torch.rand((total,), generator=gen, device=dev) * 1e-4
            s["adv"] = torch.tensor([9.0, 0.0, 0.0], device=dev)   # nine steps done
    if own:
        from tensotron_b200 import ops, runtime
        s["rt"] = ops.runtime(0)
        if case["op"].startswith("lora"):
            s["adapters"] = runtime.LoraAdapters(s["a"], s["b"], s["scale"])
        else:
            for f in ("g", "p", "m", "v"):
                if f in s:
                    s["list_" + f] = runtime.TensorList([s[f][at:at + size] for at, size in spans])
    return s


# ---- plain forms ---------------------------------------------------------------------------------------


def _chosen(idx, m, e, dev):
    """(rows, adapters): 1 where a row has that adapter."""
    if idx is None:
        return torch.zeros((m, e), device=dev).index_fill_(1, torch.zeros(1, dtype=torch.long, device=dev), 1.0)
    return (idx[:, None] == torch.arange(e, device=dev)).float()


def _down(x, a, idx):
    e, r, k = a.shape
    on = _chosen(idx, x.shape[0], e, x.device)
    return ((x @ a.reshape(e * r, k).T).view(-1, e, r) * on[:, :, None]).sum(1)


def _act_grad(dy, y, act):
    return dy * (y > 0) if act == "relu" else dy * (1 - y * y) if act == "tanh" else dy


def _plain_fwd(s, c):
    x, a, b, idx = s["x"], s["a"], s["b"], s["idx"]
    e, r, k = a.shape
    m, n = x.shape[0], b.shape[1]
    on = _chosen(idx, m, e, x.device)[:, :, None]
    wide = (x @ a.reshape(e * r, k).T).view(m, e, r) * on
    z = s["y"] if c["beside"] else x @ s["w"].T + s["bias"]
    z = z + (wide * s["scale"][:, None]).view(m, e * r) @ b.transpose(1, 2).reshape(e * r, n)
    y = torch.relu(z) if c["act"] == "relu" else torch.tanh(z) if c["act"] == "tanh" else z
    if c["beside"]:
        s["y"].copy_(y)
    return {"y": y, "t": wide.sum(1)}


def _plain_bwd(s, c):
    x, a, b, idx = s["x"], s["a"], s["b"], s["idx"]
    e, r, k = a.shape
    m, n = x.shape[0], b.shape[1]
    on = _chosen(idx, m, e, x.device)[:, :, None]
    scale = s["scale"][:, None]
    g = _act_grad(s["dy"], s["y"], c["act"])
    up = b.transpose(1, 2).reshape(e * r, n)
    dt = ((g @ up.T).view(m, e, r) * on * scale).view(m, e * r)
    dx = (s["dx"] if c["beside"] else g @ s["w"]) + dt @ a.reshape(e * r, k)
    da = (dt.T @ x).view(e, r, k)
    db = ((s["t"][:, None, :] * on * scale).view(m, e * r).T @ g).view(e, r, n).transpose(1, 2)
    if c["beside"]:
        s["dx"].copy_(dx)
    return {"dx": dx, "da": da, "db": db.contiguous()}


def _plain_norm(s):
    """The norm over the list and what the gradients are multiplied by."""
    norm = torch.stack([s["g"][at:at + size].square().sum() for at, size in s["spans"]]).sum().sqrt()
    return norm, (s["max_norm"] / (norm + CLIP_EPS)).clamp(0, 1)


def _plain_clip(s):
    norm, coef = _plain_norm(s)
    [s["g"][at:at + size].mul_(coef) for at, size in s["spans"]]
    return {"g": s["g"], "norm": norm.reshape(1)}


def _plain_adam(s):
    norm, coef = _plain_norm(s)
    s["adv"][0] += 1
    t = s["adv"][0].double()
    fix1, fix2 = (1 / (1 - BETA1 ** t)).float(), (1 / (1 - BETA2 ** t)).float()
    [_plain_adam_one(*(s[f][at:at + size] for f in "pgmv"), coef, fix1, fix2) for at, size in s["spans"]]
    return {"p": s["p"], "m": s["m"], "v": s["v"], "norm": norm.reshape(1)}


def _plain_adam_one(p, g, m, v, coef, fix1, fix2):
    g = g * coef
    m.mul_(BETA1).add_(g, alpha=1 - BETA1)
    v.mul_(BETA2).add_(g * g, alpha=1 - BETA2)
    p.sub_(LR * (m * fix1) / ((v * fix2).sqrt() + EPS))


# ---- one pass ------------------------------------------------------------------------------------------


def run(s):
    c = s["case"]
    if not own:
        return _plain_fwd(s, c) if c["op"] == "lora_fwd" else _plain_bwd(s, c) if c["op"] == "lora_bwd" else _plain_clip(s) if c["op"] == "clip" else _plain_adam(s)
    rt = s["rt"]
    if c["op"] == "lora_fwd":
        rt.LaunchLoraForward(s["adapters"], s["idx"], s["x"], s["w"], s["bias"], s["y"], s["t"], c["rows"], c["n"], c["k"], c["act"])
        return {"y": s["y"], "t": s["t"]}
    if c["op"] == "lora_bwd":
        rt.LaunchLoraBackward(s["adapters"], s["idx"], s["x"], s["w"], s["y"], s["dy"], s["t"], s["dx"], None, None, s["da"], s["db"], c["rows"], c["n"], c["k"], c["act"])
        return {"dx": s["dx"], "da": s["da"], "db": s["db"]}
    if c["op"] == "clip":
        rt.LaunchClipGradNormList(s["list_g"], s["max_norm"], CLIP_EPS, norm_out=s["norm"])
        return {"g": s["g"], "norm": s["norm"]}
    rt.LaunchClipGradNormList(s["list_g"], s["max_norm"], CLIP_EPS, norm_out=s["norm"], coef_out=s["coef"], scale=False)
    rt.LaunchAdamList(s["list_p"], s["list_g"], s["list_m"], s["list_v"], s["adv"], b1=BETA1, b2=BETA2, lr=LR, eps=EPS, grad_scale=s["coef"])
    return {"p": s["p"], "m": s["m"], "v": s["v"], "norm": s["norm"]}


def work(case):
    """Each input read once, each output written once; the adapters' tensors as far as rows can use them."""
    if not case["op"].startswith("lora"):
        n = sum(_sizes(case))
        return {"bytes": 8 * n, "flops": 3 * n} if case["op"] == "clip" else {"bytes": 28 * n, "flops": 17 * n}
    m, n, k, r, e = (case[v] for v in ("rows", "n", "k", "rank", "adapters"))
    used = min(m, e) if case["mix"] != "one" else 1
    low = r * (n + k)                      # one adapter's elements, and multiply-adds of one row through it
    rows = 0 if case["mix"] == "one" else m
    if case["op"] == "lora_fwd":
        floats = m * k + used * low + m * r + (2 * m * n if case["beside"] else n * k + n + m * n)
        return {"bytes": 4 * (floats + rows), "flops": 2 * m * (low + (0 if case["beside"] else n * k))}
    y = 0 if case["act"] == "none" else m * n
    floats = m * (k + n + r) + y + used * low + e * low + (2 * m * k if case["beside"] else n * k + m * k)
    return {"bytes": 4 * (floats + rows), "flops": 2 * m * (2 * low + (0 if case["beside"] else n * k))}


# ---- the definitions in 64 bits ------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    d = {f: v.double() for f, v in s.items() if torch.is_tensor(v) and v.is_floating_point()}
    if case["op"] in ("clip", "adam"):
        norm = torch.zeros((), dtype=torch.float64, device="cuda")
        for at, size in s["spans"]:
            norm = norm + d["g"][at:at + size].pow(2).sum()
        norm = norm.sqrt()
        coef = min(1.0, max(0.0, s["max_norm"] / (float(norm) + CLIP_EPS)))
        if case["op"] == "clip":
            for at, size in s["spans"]:
                d["g"][at:at + size] = d["g"][at:at + size] * coef
            return {"g": d["g"], "norm": norm.reshape(1)}
        t = float(s["adv"][0]) + 1
        for at, size in s["spans"]:
            w = slice(at, at + size)
            g = d["g"][w] * coef
            d["m"][w] = BETA1 * d["m"][w] + (1 - BETA1) * g
            d["v"][w] = BETA2 * d["v"][w] + (1 - BETA2) * g ** 2
            d["p"][w] = d["p"][w] - LR * (d["m"][w] / (1 - BETA1 ** t)) / (torch.sqrt(d["v"][w] / (1 - BETA2 ** t)) + EPS)
        return {"p": d["p"], "m": d["m"], "v": d["v"], "norm": norm.reshape(1)}
    m, n, k, r, e = (case[v] for v in ("rows", "n", "k", "rank", "adapters"))
    idx = torch.zeros(m, dtype=torch.long, device="cuda") if s["idx"] is None else s["idx"].long()
    of = [torch.nonzero(idx == i).flatten() for i in range(e)]
    if case["op"] == "lora_fwd":
        z = d["y"] if case["beside"] else torch.nn.functional.linear(d["x"], d["w"], d["bias"])
        t = torch.zeros((m, r), dtype=torch.float64, device="cuda")
        for i in range(e):
            t[of[i]] = torch.einsum("mk,rk->mr", d["x"][of[i]], d["a"][i])
            z[of[i]] = z[of[i]] + d["scale"][i] * torch.einsum("mr,nr->mn", t[of[i]], d["b"][i])
        return {"y": z.clamp(min=0) if case["act"] == "relu" else z.tanh() if case["act"] == "tanh" else z, "t": t}
    g = d["dy"]
    if case["act"] == "relu":
        g = torch.where(d["y"] > 0, g, torch.zeros_like(g))
    elif case["act"] == "tanh":
        g = g - g * d["y"] ** 2
    dx = d["dx"] if case["beside"] else torch.einsum("mn,nk->mk", g, d["w"])
    da, db = torch.zeros_like(d["a"]), torch.zeros_like(d["b"])
    for i in range(e):
        rows = of[i]
        dt = d["scale"][i] * torch.einsum("mn,nr->mr", g[rows], d["b"][i])
        dx[rows] = dx[rows] + torch.einsum("mr,rk->mk", dt, d["a"][i])
        da[i] = torch.einsum("mr,mk->rk", dt, d["x"][rows])
        db[i] = d["scale"][i] * torch.einsum("mn,mr->nr", g[rows], d["t"][rows])
    return {"dx": dx, "da": da, "db": db}
