"""GPU tests of the low-rank adapters (tt_lora_fwd / tt_lora_bwd, ops.LoraLinear): every output against the 64-bit
restatement within its derived elementwise bound, the masks, sizes, strides and calls where it can go wrong, and refusals."""
import numpy as np
import pytest
import torch

import adapters_ref as ref
from tensotron_b200 import ops, runtime
from tensotron_b200.runtime import ACT, LoraAdapters, TensorRuntime, TensotronGemmError

pytestmark = pytest.mark.gpu

GUARD = 64


def dev(v, offset=0):
    """A CUDA copy; with an offset, a view that starts `offset` floats behind an aligned address."""
    if v is None:
        return None
    t = torch.from_numpy(np.ascontiguousarray(v))
    if not offset:
        return t.cuda()
    buf = torch.empty(t.numel() + offset, dtype=t.dtype, device="cuda")
    buf[offset:].copy_(t.reshape(-1))
    return buf[offset:].view(t.shape)


class Out:
    """An output between guard words that must stay as they are."""

    def __init__(self, shape, fill=None, offset=0):
        n = int(np.prod(shape))
        self.buf = torch.full((n + 2 * GUARD + offset,), 7.5, device="cuda")
        self.t = self.buf[GUARD + offset:GUARD + offset + n].view(shape)
        self.t.copy_(torch.from_numpy(fill)) if fill is not None else self.t.fill_(float("nan"))
        self.lo, self.hi = GUARD + offset, GUARD + offset + n

    def get(self):
        assert bool((self.buf[:self.lo] == 7.5).all()) and bool((self.buf[self.hi:] == 7.5).all()), "wrote outside the output"
        return self.t.cpu().numpy().astype(np.float64)


def near(got, want, bound, name):
    assert got.shape == want.shape
    off = np.abs(got - want)
    bad = ~(off <= bound)
    assert not bad.any(), "%s: %d of %d outside, worst %.3g against bound %.3g" % (
        name, bad.sum(), bad.size, off[bad].max(), bound[bad].max())


def run_fwd(rt, d, kind, proj, want_t=True, offset=0):
    m, k = d["x"].shape
    e, n, r = d["b"].shape
    ad = LoraAdapters(dev(d["a"], offset), dev(d["b"], offset), dev(d["s"]))
    y = Out((m, n), None if proj else d["y"], offset)
    t = Out((m, r), None, offset) if want_t else None
    rt.LaunchLoraForward(ad, dev(d["idx"]), dev(d["x"], offset), dev(d["w"], offset) if proj else None, dev(d["bias"], offset) if proj else None,
                         y.t, t.t if want_t else None, m, n, k, kind)
    rt.Check()
    return y.get(), t.get() if want_t else None


# Few rows: w cut over 4 and 8 CTAs along k, more outputs than one pass of the SMs takes (also odd ones), a k that does not
# fit and goes to the tiles, one row more than that form takes
FEW_ROWS = [(16, 64, 8192, 8, 3), (13, 100, 16384, 4, 3), (9, 24, 20000, 4, 2), (3, 40, 20000, 16, 5), (1, 8, 40000, 4, 2), (4, 10000, 128, 8, 3),
            (2, 20011, 64, 6, 3), (5, 9001, 33, 3, 2), (64, 300, 260, 16, 9), (65, 300, 260, 16, 9), (33, 777, 1028, 128, 4), (48, 4096, 516, 2, 60)]


@pytest.mark.parametrize("proj", [True, False])
@pytest.mark.parametrize("shape", FEW_ROWS)
def test_forward_of_few_rows(rt, shape, proj):
    m, n, k, r, e = shape
    kind = ["none", "relu", "tanh"][(m + n) % 3]
    d = ref.inputs(m * 7 + r, m, n, k, r, e, "mixed")
    y, t, ey, et = ref.forward(d["x"], d["w"] if proj else None, d["bias"], d["a"], d["b"], d["s"], d["idx"], kind, d["y"])
    gy, gt = run_fwd(rt, d, kind, proj)
    near(gt, t, et, "t")
    near(gy, y, ey, "y")
    again = run_fwd(rt, d, kind, proj)
    assert np.array_equal(gy, again[0]) and np.array_equal(gt, again[1])


# rows, n, k, rank, adapters: single tokens, few rows, one row more and less than a tile, odd sizes, ranks between the
# kernels' widths and the highest, more adapters than rows, narrow and long contractions
SHAPES = [(1, 64, 64, 4, 3), (1, 1, 1, 1, 1), (2, 5, 3, 2, 1), (5, 33, 17, 1, 2), (16, 256, 512, 16, 40), (17, 130, 260, 8, 4),
          (63, 64, 128, 4, 1), (65, 127, 129, 5, 3), (64, 64, 128, 4, 1), (130, 257, 100, 7, 5), (333, 517, 1000, 6, 5),
          (200, 128, 256, 64, 3), (100, 130, 70, 100, 4), (96, 132, 64, 128, 2), (300, 96, 4096, 16, 40), (700, 512, 36, 33, 7),
          (1030, 36, 516, 12, 200), (700, 36, 40, 3, 600), (300, 16, 24, 2, 4096)]


@pytest.mark.parametrize("mix", ["mixed", "one", "sorted", "last", "none"])
@pytest.mark.parametrize("proj", [True, False])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(rt, shape, proj, mix):
    m, n, k, r, e = shape
    kind = ["none", "relu", "tanh"][(m + n) % 3]
    d = ref.inputs(hash(shape) % 10000, m, n, k, r, e, mix)
    y, t, ey, et = ref.forward(d["x"], d["w"] if proj else None, d["bias"], d["a"], d["b"], d["s"], d["idx"], kind, d["y"])
    gy, gt = run_fwd(rt, d, kind, proj)
    near(gt, t, et, "t")
    near(gy, y, ey, "y")


def run_bwd(rt, d, kind, proj, t, base=True, give_t=True, offset=0):
    m, k = d["x"].shape
    e, n, r = d["b"].shape
    ad = LoraAdapters(dev(d["a"], offset), dev(d["b"], offset), dev(d["s"]))
    o = dict(dx=Out((m, k), None if proj else d["dx"], offset), da=Out((e, r, k), None, offset), db=Out((e, n, r), None, offset))
    if proj and base:
        o.update(dw=Out((n, k), None, offset), dbias=Out((n,), None, offset))
    rt.LaunchLoraBackward(ad, dev(d["idx"]), dev(d["x"], offset), dev(d["w"], offset) if proj else None, dev(d["y"], offset), dev(d["dy"], offset),
                          dev(t, offset) if give_t else None, o["dx"].t, o["dw"].t if "dw" in o else None,
                          o["dbias"].t if "dbias" in o else None, o["da"].t, o["db"].t, m, n, k, kind)
    rt.Check()
    return {name: v.get() for name, v in o.items()}


@pytest.mark.parametrize("mix", ["mixed", "one", "sorted", "last", "none"])
@pytest.mark.parametrize("proj", [True, False])
@pytest.mark.parametrize("shape", SHAPES)
def test_backward(rt, shape, proj, mix):
    m, n, k, r, e = shape
    kind = ["none", "relu", "tanh"][(m + k) % 3]
    d = ref.inputs(hash(shape) % 10000 + 1, m, n, k, r, e, mix)
    if kind == "tanh":
        d["y"] = np.tanh(d["y"])
    t = ref.forward(d["x"], None, None, d["a"], d["b"], d["s"], d["idx"], kind, d["y"])[1].astype(np.float32)
    want = ref.backward(d["x"], d["w"] if proj else None, d["a"], d["b"], d["s"], d["idx"], kind, d["y"], d["dy"], t, d["dx"])
    for base in ([True, False] if proj else [False]):        # (without the projection's gradients small layers take one launch)
        got = run_bwd(rt, d, kind, proj, t, base)
        for name, v in got.items():
            near(v, *want[name], name)


# the one-launch form's limits (rows, outputs, rows x N, rows x rank, rank, adapters, adapters x N x rank, adapters x rank,
# rows x N x K), and one beyond each
SMALL = [(64, 64, 128, 4, 1), (256, 32, 256, 16, 2), (256, 32, 255, 8, 16), (32, 256, 256, 2, 16), (33, 248, 33, 5, 6), (1, 256, 1000, 16, 2), (7, 200, 299, 3, 13),
         (256, 1, 31, 8, 3), (257, 8, 16, 4, 2), (20, 257, 16, 4, 2), (64, 129, 64, 4, 2), (64, 64, 64, 17, 2), (32, 32, 64, 4, 17), (8, 256, 16, 11, 3), (8, 16, 16, 13, 10),
         (64, 64, 513, 4, 2)]


@pytest.mark.parametrize("mix", ["mixed", "one", "none"])
@pytest.mark.parametrize("proj", [True, False])
@pytest.mark.parametrize("shape", SMALL)
def test_backward_of_small_layers(rt, shape, proj, mix):
    m, n, k, r, e = shape
    kind = ["none", "relu", "tanh"][(n + k) % 3]
    d = ref.inputs(m + 3 * k, m, n, k, r, e, mix)
    if kind == "tanh":
        d["y"] = np.tanh(d["y"])
    t = ref.forward(d["x"], None, None, d["a"], d["b"], d["s"], d["idx"], kind, d["y"])[1].astype(np.float32)
    want = ref.backward(d["x"], d["w"] if proj else None, d["a"], d["b"], d["s"], d["idx"], kind, d["y"], d["dy"], t, d["dx"])
    rt.ResetCounters()
    got = run_bwd(rt, d, kind, proj, t, base=False)
    if not proj and mix == "mixed":
        small = (m <= 256 and n <= 256 and r <= 16 and e <= 16 and m * n <= 8192 and m * r <= 4096 and e * n * r <= 8192 and
                 e * r <= 128 and m * n * k <= 1 << 21)
        assert (rt.Stats()["launches"] == 1) == small
    for name, v in got.items():
        near(v, *want[name], name)
    again = run_bwd(rt, d, kind, proj, t, base=False)
    assert all(np.array_equal(got[f], again[f]) for f in got)


@pytest.mark.parametrize("offset", [1, 2, 3])
def test_unaligned_views_and_no_t(rt, offset):
    d = ref.inputs(5, 70, 64, 96, 8, 3, "mixed")
    y, t, ey, et = ref.forward(d["x"], d["w"], d["bias"], d["a"], d["b"], d["s"], d["idx"], "relu")
    gy, _ = run_fwd(rt, d, "relu", True, want_t=False, offset=offset)
    near(gy, y, ey, "y")
    d["y"] = y.astype(np.float32)
    want = ref.backward(d["x"], d["w"], d["a"], d["b"], d["s"], d["idx"], "relu", d["y"], d["dy"], t)
    got = run_bwd(rt, d, "relu", True, None, give_t=False, offset=offset)
    for name, v in got.items():
        bound = want[name][1]
        if name == "db":            # t is recomputed here, so its own error comes in
            for i, rows in enumerate(ref.rows_of(d["idx"], 70, 3)):
                bound[i] += d["s"][i] * (np.abs(ref.act_grad(d["dy"], d["y"], "relu")[rows]).T @ et[rows])
        near(v, want[name][0], bound, name)


def test_every_gradient_can_be_left_out(rt):
    d = ref.inputs(6, 40, 48, 32, 4, 3, "mixed")
    t = ref.forward(d["x"], d["w"], d["bias"], d["a"], d["b"], d["s"], d["idx"], "none")[1].astype(np.float32)
    want = ref.backward(d["x"], d["w"], d["a"], d["b"], d["s"], d["idx"], "none", d["y"], d["dy"], t)
    ad = LoraAdapters(dev(d["a"]), dev(d["b"]), dev(d["s"]))
    shapes = dict(dx=(40, 32), dw=(48, 32), dbias=(48,), da=(3, 4, 32), db=(3, 48, 4))
    for name in list(shapes) + [None]:
        o = {f: Out(shapes[f]) if f == name else None for f in shapes}
        x = dev(d["x"]) if name in ("dw", "da") else None        # not read otherwise
        rt.LaunchLoraBackward(ad, dev(d["idx"]), x, dev(d["w"]), None, dev(d["dy"]), dev(t) if name == "db" else None,
                              *[o[f].t if o[f] else None for f in ("dx", "dw", "dbias", "da", "db")], 40, 48, 32, "none")
        rt.Check()
        if name:
            near(o[name].get(), *want[name], name)


def test_no_scale_means_one(rt):
    d = ref.inputs(7, 33, 40, 24, 4, 2, "mixed")
    d["s"] = np.ones(2, np.float32)
    ad = LoraAdapters(dev(d["a"]), dev(d["b"]))
    y, _, ey, _ = ref.forward(d["x"], d["w"], None, d["a"], d["b"], d["s"], d["idx"], "none")
    out = Out((33, 40))
    rt.LaunchLoraForward(ad, dev(d["idx"]), dev(d["x"]), dev(d["w"]), None, out.t, None, 33, 40, 24)
    near(out.get(), y, ey, "y")


def test_no_rows(rt):
    f = lambda *s: torch.full(s, 3.0, device="cuda")     # noqa: E731
    ad = LoraAdapters(f(2, 4, 8), f(2, 6, 4))
    idx = torch.zeros(5, dtype=torch.int32, device="cuda")
    da, db, dw, dbias, y = f(2, 4, 8), f(2, 6, 4), f(6, 8), f(6), f(5, 6)
    rt.LaunchLoraBackward(ad, idx, f(1, 8), f(6, 8), None, f(1, 6), None, f(1, 8), dw, dbias, da, db, 0, 6, 8)
    rt.LaunchLoraForward(ad, idx, f(1, 8), f(6, 8), None, y, None, 0, 6, 8)
    rt.Check()
    assert all(bool((v == 0).all()) for v in (da, db, dw, dbias)) and bool((y == 3).all())


def test_bad_indices_are_reported_and_never_used(rt):
    d = ref.inputs(8, 80, 32, 48, 4, 3, "mixed")
    bad = d["idx"].copy()
    for at, v in ((0, 3), (17, -2), (63, 2 ** 31 - 1), (79, -2 ** 31)):
        d["idx"][at], bad[at] = -1, v
    y, t, ey, et = ref.forward(d["x"], d["w"], d["bias"], d["a"], d["b"], d["s"], d["idx"], "none")
    ad = LoraAdapters(dev(d["a"]), dev(d["b"]), dev(d["s"]))
    oy, ot = Out((80, 32)), Out((80, 4))
    rt.LaunchLoraForward(ad, dev(bad), dev(d["x"]), dev(d["w"]), dev(d["bias"]), oy.t, ot.t, 80, 32, 48)
    with pytest.raises(TensotronGemmError) as err:
        rt.Check()
    assert err.value.status == 8
    near(oy.get(), y, ey, "y")
    near(ot.get(), t, et, "t")
    rt.Check()                                      # the report was taken back
    want = ref.backward(d["x"], d["w"], d["a"], d["b"], d["s"], d["idx"], "none", d["y"], d["dy"], t)
    for part in (dict(da=Out((3, 4, 48)), db=Out((3, 32, 4))), dict(dx=Out((80, 48)), dw=Out((32, 48)))):     # in one launch, and in several
        rt.LaunchLoraBackward(ad, dev(bad), dev(d["x"]), dev(d["w"]), None, dev(d["dy"]), dev(t.astype(np.float32)),
                              *[part[f].t if f in part else None for f in ("dx", "dw", "dbias", "da", "db")], 80, 32, 48)
        with pytest.raises(TensotronGemmError) as err:
            rt.Check()
        assert err.value.status == 8
        for name, v in part.items():
            near(v.get(), *want[name], name)


@pytest.mark.parametrize("m,n,k", [(150, 70, 90), (60, 70, 90), (14, 33, 50)])
def test_not_finite_values_stay_with_their_rows_and_adapters(rt, m, n, k):
    """A NaN in one adapter reaches its own rows and gradients only; an infinite row its own outputs and its adapter's
    gradients only; rows without an adapter meet none of it."""
    d = ref.inputs(9, m, n, k, 6, 4, "mixed")
    d["idx"][:4] = [2, 1, -1, 0]
    d["a"][1, 2, 3] = np.nan
    d["b"][1, 4, 2] = np.nan
    row = int(np.nonzero(d["idx"] == 2)[0][0])
    d["x"][row, 5] = np.inf
    d["dy"][row, 1] = np.inf
    clean = (d["idx"] != 1)
    clean[row] = False
    y, t = run_fwd(rt, d, "none", True)
    assert np.isfinite(y[clean]).all() and np.isfinite(t[clean]).all()
    assert np.isnan(y[d["idx"] == 1]).all() and not np.isfinite(y[row]).any()
    got = run_bwd(rt, d, "none", True, np.nan_to_num(t, posinf=1.0, neginf=-1.0).astype(np.float32), base=False)
    assert np.isfinite(got["dx"][clean]).all() and np.isnan(got["dx"][d["idx"] == 1]).all()
    for e in (0, 3):
        assert np.isfinite(got["da"][e]).all() and np.isfinite(got["db"][e]).all()
    assert np.isnan(got["da"][1][2]).all() and not np.isfinite(got["db"][2][1]).any()


def test_repeats_are_bitwise_and_leave_inputs_alone(rt):
    d = ref.inputs(10, 500, 264, 300, 16, 9, "mixed")
    first, second = run_fwd(rt, d, "tanh", True), run_fwd(rt, d, "tanh", True)
    assert all(np.array_equal(p, q) for p, q in zip(first, second))
    t = first[1].astype(np.float32)
    d["y"] = first[0].astype(np.float32)
    one, two = run_bwd(rt, d, "tanh", True, t), run_bwd(rt, d, "tanh", True, t)
    assert all(np.array_equal(one[f], two[f]) for f in one)


def test_row_order_does_not_change_a_rows_output(rt):
    """The same rows in another order give the same bits, row by row (the grouping is stable, a row's sums are its own)."""
    d = ref.inputs(11, 260, 128, 192, 8, 5, "mixed")
    p = np.random.default_rng(0).permutation(260)
    y, t = run_fwd(rt, d, "none", True)
    d["x"], d["idx"] = d["x"][p], d["idx"][p]
    y2, t2 = run_fwd(rt, d, "none", True)
    assert np.array_equal(y[p], y2) and np.array_equal(t[p], t2)


@pytest.mark.parametrize("m", [3, 200])
def test_captured_calls_follow_new_row_adapters(rt, m):
    """A captured forward + backward replays with other rows, other adapters per row and other values in the same buffers."""
    n, k, r, e = 72, 60, 8, 5
    d = ref.inputs(12, m, n, k, r, e, "mixed")
    ad = LoraAdapters(dev(d["a"]), dev(d["b"]), dev(d["s"]))
    buf = {f: dev(d[f]) for f in ("x", "w", "bias", "dy", "idx")}
    y, t, dx, da, db = (torch.zeros(s, device="cuda") for s in ((m, n), (m, r), (m, k), (e, r, k), (e, n, r)))

    def call():
        rt.LaunchLoraForward(ad, buf["idx"], buf["x"], buf["w"], buf["bias"], y, t, m, n, k, "relu")
        rt.LaunchLoraBackward(ad, buf["idx"], buf["x"], buf["w"], y, buf["dy"], t, dx, None, None, da, db, m, n, k, "relu")

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for seed, mix in ((13, "mixed"), (14, "last"), (15, "none"), (16, "sorted")):
        q = ref.inputs(seed, m, n, k, r, e, mix)
        for f in buf:
            if f != "w":
                buf[f].copy_(torch.from_numpy(q[f]))
        graph.replay()
        rt.Check()
        q.update(w=d["w"], a=d["a"], b=d["b"], s=d["s"])
        wy, wt, ey, et = ref.forward(q["x"], q["w"], q["bias"], q["a"], q["b"], q["s"], q["idx"], "relu")
        gy, gt = y.cpu().numpy(), t.cpu().numpy()
        near(gy.astype(np.float64), wy, ey, "y")
        near(gt.astype(np.float64), wt, et, "t")
        want = ref.backward(q["x"], q["w"], q["a"], q["b"], q["s"], q["idx"], "relu", gy, q["dy"], gt)
        for name, v in (("dx", dx), ("da", da), ("db", db)):
            near(v.cpu().numpy().astype(np.float64), *want[name], name)


def test_two_handles_on_two_streams(rt):
    other = TensorRuntime(0, 64 << 20)
    d1, d2 = ref.inputs(20, 300, 200, 256, 16, 6, "mixed"), ref.inputs(21, 40, 200, 256, 16, 6, "mixed")
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    todo = []
    for d in (d1, d2):
        m = d["x"].shape[0]
        todo.append((LoraAdapters(dev(d["a"]), dev(d["b"]), dev(d["s"])), dev(d["idx"]), dev(d["x"]), dev(d["w"]), dev(d["bias"]),
                     torch.empty((m, 200), device="cuda"), torch.empty((m, 16), device="cuda"), m))
    torch.cuda.synchronize()
    for _ in range(20):
        for r, st, q in zip((rt, other), streams, todo):
            r.LaunchLoraForward(*q[:7], q[7], 200, 256, "none", stream=st)
    torch.cuda.synchronize()
    for d, q in zip((d1, d2), todo):
        y, _, ey, _ = ref.forward(d["x"], d["w"], d["bias"], d["a"], d["b"], d["s"], d["idx"], "none")
        near(q[5].cpu().numpy().astype(np.float64), y, ey, "y")
    other.Dispose()


def test_refusals(rt):
    f = lambda *s: torch.zeros(s, device="cuda")     # noqa: E731
    ad = LoraAdapters(f(2, 4, 8), f(2, 6, 4))
    ok = dict(adapters=ad, row_adapter=None, x=f(3, 8), w=f(6, 8), bias=None, y=f(3, 6), t=None, M=3, N=6, K=8)

    def status(**change):
        with pytest.raises(TensotronGemmError) as err:
            rt.LaunchLoraForward(**{**ok, **change})
        return err.value.status

    rt.LaunchLoraForward(**ok)
    assert status(M=-1) == 1 and status(N=0) == 1 and status(K=0) == 1 and status(x=None) == 1 and status(y=None) == 1
    assert status(w=None, bias=f(6)) == 1
    assert status(row_adapter=torch.zeros(3, dtype=torch.int64, device="cuda")) == 1
    with pytest.raises(KeyError):
        rt.LaunchLoraForward(**{**ok, "act": "gelu"})
    assert status(adapters=LoraAdapters(f(1, 129, 8), f(1, 6, 129))) == 3
    assert status(adapters=LoraAdapters(f(4097, 1, 1), f(4097, 6, 1))) == 3
    assert status(M=1 << 20, N=1 << 12) == 3                    # offsets beyond int32
    assert status(M=0, N=2 ** 31 - 1) == 3 and status(M=0, K=2 ** 31 - 1) == 3
    tiny = TensorRuntime(0, 4096)
    with pytest.raises(TensotronGemmError) as err:
        tiny.LaunchLoraForward(**{**ok, "x": f(2000, 8), "y": f(2000, 6), "M": 2000})
    assert err.value.status == 4
    tiny.Dispose()
    back = [ad, None, f(3, 8), f(6, 8), None, f(3, 6), None, f(3, 8), None, None, f(2, 4, 8), f(2, 6, 4), 3, 6, 8]
    rt.LaunchLoraBackward(*back)
    for at, v, extra in ((5, None, {}), (2, None, {}), (3, None, {8: f(6, 8)}), (3, None, {9: f(6)})):
        args = list(back)
        args[at] = v
        for i, q in extra.items():
            args[i] = q
        with pytest.raises(TensotronGemmError) as err:
            rt.LaunchLoraBackward(*args)
        assert err.value.status == 1
    with pytest.raises(TensotronGemmError) as err:
        rt.LaunchLoraBackward(*back, "relu")                    # needs y
    assert err.value.status == 1
    for a, b, s in ((f(2, 4, 8), f(3, 6, 4), None), (f(2, 4, 8), f(2, 6, 5), None), (f(2, 4), f(2, 6, 4), None), (f(2, 4, 8), f(2, 6, 4), f(3))):
        with pytest.raises(ValueError):
            LoraAdapters(a, b, s)
    with pytest.raises(TypeError):
        LoraAdapters(f(2, 4, 8).double(), f(2, 6, 4))
    with pytest.raises(TypeError):
        LoraAdapters(f(2, 8, 4).transpose(1, 2), f(2, 6, 4))


@pytest.mark.parametrize("mode", [runtime.TT_MATH_TF32, runtime.TT_MATH_3XTF32])
def test_math_mode_reaches_the_projection_only(rt, mode):
    """The projection follows the handle's mode (TF32: inputs cut to 10 mantissa bits, 2^-10 relative each; the 3xTF32 bound
    is the strict one plus the accumulator's (3K/8) 2^-23); t is strict FP32 in every mode."""
    m, n, k = 512, 512, 1024
    d = ref.inputs(30, m, n, k, 16, 4, "mixed")
    y, t, ey, et = ref.forward(d["x"], d["w"], d["bias"], d["a"], d["b"], d["s"], d["idx"], "none")
    mass = np.abs(d["x"].astype(np.float64)) @ np.abs(d["w"].astype(np.float64)).T
    rt.SetCuBlasMathMode(mode)
    try:
        gy, gt = run_fwd(rt, d, "none", True)
    finally:
        rt.SetCuBlasMathMode(runtime.TT_MATH_FP32)
    near(gt, t, et, "t")
    extra = 2.1 * 2.0 ** -10 * mass if mode == runtime.TT_MATH_TF32 else 2.0 ** -20 * mass
    near(gy, y, ey + extra + (3 * k / 8) * 2.0 ** -23 * mass, "y")


def test_lora_linear_layer(rt):
    gen = torch.Generator().manual_seed(0)
    lin = ops.LoraLinear(96, 80, rank=8, adapters=4, alpha=16, act="tanh", generator=gen)
    assert lin.Scale.tolist() == [2.0] * 4 and bool((lin.B == 0).all())
    x = torch.randn((50, 96), generator=gen).cuda()
    idx = torch.randint(-1, 4, (50,), generator=gen).to(torch.int32).cuda()
    y0, _ = lin.Forward(x, idx)
    plain = ops.Linear.Forward(lin, x)
    # B = 0: the projection alone, through another kernel's summation order
    assert torch.allclose(y0, plain, atol=1e-5)
    lin.B = torch.randn((4, 80, 8), generator=gen).cuda() * 0.3         # replaced, not written in place
    y, t = lin.Forward(x, idx)
    dy = torch.randn((50, 80), generator=gen).cuda()
    grads = dict(zip(("dx", "da", "db", "dw", "dbias"), lin.Backward(x, y, t, dy, idx, need_base=True)))
    rt.Check()
    h = lambda v: v.cpu().numpy()       # noqa: E731
    args = [h(v) for v in (x, lin.Weight, lin.A, lin.B, lin.Scale, idx)]
    wy, _, ey, _ = ref.forward(args[0], args[1], h(lin.Bias), *args[2:], "tanh")
    near(h(y).astype(np.float64), wy, ey, "y")
    want = ref.backward(*args, "tanh", h(y), h(dy), h(t))
    for name, v in grads.items():
        near(h(v).astype(np.float64), *want[name], name)
    assert lin.Backward(x, y, None, dy, idx, need_dx=False)[0] is None
    for bad in (dict(x=x[:, :95].contiguous()), dict(row_adapter=idx.long()), dict(row_adapter=idx[:49])):
        with pytest.raises(TensotronGemmError):
            lin.Forward(**{"x": x, "row_adapter": idx, **bad})
    with pytest.raises(TensotronGemmError):
        lin.Backward(x, y, t[:, :7].contiguous(), dy, idx)


def test_adapter_training_step_end_to_end(rt):
    """The operators as a program uses them: a layer's adapters through the loss, their gradients, the clipped step over the
    list of adapter tensors -- against the same step in 64 bits."""
    gen = torch.Generator().manual_seed(3)
    lin = ops.LoraLinear(64, 10, rank=4, adapters=3, alpha=8, generator=gen)
    lin.B = (torch.randn((3, 10, 4), generator=gen) * 0.2).cuda()
    x = torch.randn((90, 64), generator=gen).cuda()
    idx = torch.randint(0, 3, (90,), generator=gen).to(torch.int32).cuda()
    labels = torch.randint(0, 10, (90,), generator=gen).to(torch.int32).cuda()
    a, b = lin.A.double().cpu().numpy(), lin.B.double().cpu().numpy()
    opt = ops.Adam([lin.A, lin.B], lr=1e-2)
    y, t = lin.Forward(x, idx)
    dl, loss = torch.empty_like(y), torch.zeros(1, device="cuda")
    rt.LaunchSoftmaxCrossEntropy(y, labels, dl, loss, 90, 10, 1.0 / 90)
    _, da, db, _, _ = lin.Backward(x, y, t, dl, idx, need_dx=False)
    norm = opt.Step([da, db], max_norm=0.05)
    rt.Check()
    h = lambda v: v.double().cpu().numpy()       # noqa: E731
    wy, wt, _, _ = ref.forward(h(x), h(lin.Weight), h(lin.Bias), a, b, h(lin.Scale), idx.cpu().numpy(), "none")
    p = np.exp(wy - wy.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    lab = labels.cpu().numpy()
    assert abs(loss.item() + np.log(p[np.arange(90), lab]).mean()) < 1e-5
    p[np.arange(90), lab] -= 1
    want = ref.backward(h(x), h(lin.Weight), a, b, h(lin.Scale), idx.cpu().numpy(), "none", wy, p / 90, wt)
    wn, coef = ref.clip([want["da"][0], want["db"][0]], 0.05, 1e-6)
    assert abs(norm.item() - wn) <= 1e-5 * wn and coef < 1
    for p0, g, got, mom in ((a, want["da"][0], lin.A, opt.M.tensors[0]), (b, want["db"][0], lin.B, opt.M.tensors[1])):
        q, m, _ = ref.adam(p0, g, np.zeros_like(g), np.zeros_like(g), 1, coef, lr=1e-2)
        # the first step moves a weight by lr * g / (|g| + eps'): its sign decides, so weights whose gradient is within the
        # gradients' error of zero are left out of the comparison, and the moments are compared everywhere
        np.testing.assert_allclose(h(mom), m, atol=1e-6 * np.abs(m).max() + 1e-9, rtol=1e-4)
        clear = np.abs(g) > 1e-3 * np.abs(g).max()
        assert clear.mean() > 0.5
        np.testing.assert_allclose(h(got)[clear], q[clear], atol=1e-5)


def test_offsets_close_to_int32(rt):
    """x and dx of almost 2^31 elements: the last rows' offsets only just fit an int32."""
    m, n, k, r, e = 524287, 8, 4096, 2, 3
    gen = torch.Generator(device="cuda").manual_seed(1)
    f = lambda *s: torch.randn(s, generator=gen, device="cuda")      # noqa: E731
    x, dx, dy, a, b = f(m, k), f(m, k), f(m, n), f(e, r, k) / 64, f(e, n, r)
    idx = torch.randint(-1, e, (m,), generator=gen, device="cuda").to(torch.int32)
    ad = LoraAdapters(a, b)
    t, y, da, dx0 = torch.empty((m, r), device="cuda"), torch.zeros((m, n), device="cuda"), torch.empty_like(a), dx[-300:].clone()
    rt.LaunchLoraForward(ad, idx, x, None, None, y, t, m, n, k)
    rt.LaunchLoraBackward(ad, idx, x, None, None, dy, None, dx, None, None, da, None, m, n, k)
    rt.Check()
    last = slice(m - 300, m)
    h = lambda v: v.double().cpu().numpy()       # noqa: E731
    args = [h(x[last]), None, None, h(a), h(b), np.ones(e), idx[last].cpu().numpy(), "none", np.zeros((300, n))]
    wy, wt, ey, et = ref.forward(*args)
    near(h(y[last]), wy, ey, "y")
    near(h(t[last]), wt, et, "t")
    want = ref.backward(args[0], None, h(a), h(b), np.ones(e), args[6], "none", np.zeros((300, n)), h(dy[last]), wt, h(dx0))
    near(h(dx[last]), *want["dx"], "dx")
    # dA over all rows: the same products added in 64 bits, against (count + 32) roundings of their absolute sum
    sums, mass = torch.zeros((e, r, k), dtype=torch.float64, device="cuda"), torch.zeros((e, r, k), dtype=torch.float64, device="cuda")
    for at in range(0, m, 32768):
        rows = slice(at, min(m, at + 32768))
        for i in range(e):
            on = (idx[rows] == i).double()[:, None]
            dt = (dy[rows].double() @ b[i].double()) * on
            sums[i] += dt.T @ x[rows].double()
            mass[i] += ((dy[rows].double().abs() @ b[i].double().abs()) * on).T @ x[rows].double().abs()
    near(h(da), h(sums), (m + 32) * ref.U * h(mass), "da")
    # (that bound is loose at this count: the error of a sum of random signs grows with the root of it)
    assert float((da - sums).norm() / sums.norm()) < m ** 0.5 * ref.U
