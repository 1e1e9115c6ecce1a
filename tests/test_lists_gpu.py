"""GPU tests of ClipGradNorm and Adam over lists of tensors (tt_clip_grad_norm_list, tt_adam_step_list, ops.ClipGradNorm,
ops.Adam) against the 64-bit restatement."""
import numpy as np
import pytest
import torch

import adapters_ref as ref
from tensotron_b200 import ops
from tensotron_b200.runtime import TensorList, TensorRuntime, TensotronGemmError

pytestmark = pytest.mark.gpu
U = 2.0 ** -24

# single values, empty tensors, sizes around the vector width and the chunk, more tensors than one table holds
LISTS = {"one value": [1], "empty tensors": [0, 5, 0, 0, 3, 0], "nothing": [], "only empty": [0, 0],
         "control net": [512, 64, 4096, 64, 128, 2], "chunk edges": [4095, 4096, 4097, 8191, 8192, 8193, 3],
         "many": [(i * 37) % 300 for i in range(1500)], "two": [1 << 20, 3], "large": [3_000_001, 1_000_003, 17]}


def tensors(sizes, seed, pack, scale=1.0):
    """Tensors of one flat buffer; pack: no alignment between them, and an odd start."""
    at, spans = (1 if pack else 0), []
    for n in sizes:
        spans.append((at, n))
        at += n if pack else -(-n // 4) * 4
    rng = np.random.default_rng(seed)
    flat = torch.from_numpy((rng.standard_normal(at + 8) * scale).astype(np.float32)).cuda()
    return flat, [flat[o:o + n] for o, n in spans]


@pytest.mark.parametrize("pack", [False, True])
@pytest.mark.parametrize("name", list(LISTS))
@pytest.mark.parametrize("share", [0.5, 2.0])
def test_clip(rt, name, pack, share):
    """share: max_norm over the norm; above 1 nothing is clipped, and the gradients keep their bits."""
    flat, ts = tensors(LISTS[name], 1, pack)
    before, gs = flat.clone(), [t.cpu().numpy().copy() for t in ts]
    norm, _ = ref.clip(gs, 1.0, 0.0)
    max_norm = max(norm, 1.0) * share
    _, coef = ref.clip(gs, max_norm, 1e-6)
    out = torch.full((2,), float("nan"), device="cuda")
    rt.LaunchClipGradNormList(ts, max_norm, 1e-6, norm_out=out[:1], coef_out=out[1:])
    rt.Check()
    # double sums: the norm is rounded once; the coefficient adds a sum, a quotient and the rounding of max_norm and eps
    assert abs(out[0].item() - norm) <= 2 * U * norm
    assert abs(out[1].item() - coef) <= 6 * U * coef
    for t, g in zip(ts, gs):
        assert np.all(np.abs(t.cpu().numpy() - coef * g.astype(np.float64)) <= 8 * U * coef * np.abs(g) + 1e-45)
    inside = torch.zeros_like(flat, dtype=torch.bool)
    for t in ts:
        inside[t.storage_offset():t.storage_offset() + t.numel()] = True
    assert torch.equal(flat[~inside], before[~inside])          # nothing between and behind the tensors was touched
    if share > 1:
        assert torch.equal(flat, before)
    # the same call again on the same values: the same bits
    again = before.clone()
    rt.LaunchClipGradNormList([again[t.storage_offset():t.storage_offset() + t.numel()] for t in ts], max_norm, 1e-6)
    assert torch.equal(again, flat)


def test_norm_alone_leaves_the_gradients(rt):
    flat, ts = tensors([1000, 50000, 7], 2, False)
    before = flat.clone()
    out = torch.zeros(2, device="cuda")
    rt.LaunchClipGradNormList(TensorList(ts), 1.0, norm_out=out[:1], coef_out=out[1:], scale=False)
    rt.Check()
    norm, coef = ref.clip([t.cpu().numpy() for t in ts], 1.0, 1e-6)
    assert torch.equal(flat, before) and abs(out[0].item() - norm) <= 2 * U * norm and abs(out[1].item() - coef) <= 6 * U * coef


def test_extreme_gradients(rt):
    """Squares of these overflow or vanish in float32; not their sum in 64 bits."""
    for big in (1e30, 1e-30):
        ts = [torch.full((n,), big, device="cuda") for n in (100, 5000)]
        norm = ops.ClipGradNorm(ts, big)
        assert abs(norm.item() - big * 5100 ** 0.5) <= 4 * U * big * 5100 ** 0.5
        if big > 1:
            assert abs(ts[0][0].item() - big / 5100 ** 0.5) <= 8 * U * big
    # infinite: coefficient 0 (an infinite gradient becomes NaN, the finite ones 0); NaN reaches everything
    ts = [torch.ones(10, device="cuda"), torch.ones(5000, device="cuda")]
    ts[1][77] = float("inf")
    assert ops.ClipGradNorm(ts, 1.0).item() == float("inf")
    assert bool((ts[0] == 0).all()) and int(torch.isnan(ts[1]).sum()) == 1 and int((ts[1] == 0).sum()) == 4999
    ts = [torch.ones(10, device="cuda"), torch.ones(5000, device="cuda")]
    ts[0][3] = float("nan")
    assert np.isnan(ops.ClipGradNorm(ts, 1.0).item())
    assert all(bool(torch.isnan(t).all()) for t in ts)
    # max_norm 0 and below: everything becomes 0
    for limit in (0.0, -1.0):
        ts = [torch.ones(300, device="cuda")]
        ops.ClipGradNorm(ts, limit)
        assert bool((ts[0] == 0).all())
    zero = [torch.zeros(300, device="cuda")]
    assert ops.ClipGradNorm(zero, 1.0).item() == 0 and bool((zero[0] == 0).all())


def adam_bound(p, g, m, v, t, coef, lr, b1, b2):
    """Elementwise bounds of a float32 step: m and v are two products and a sum, the update a handful of roundings of
    lr * m' / sqrt(v'); the bias corrections' powf is off by a few units and 1 - b^t loses log2(1 / (1 - b^t)) bits."""
    m1, v1 = np.abs(b1 * m) + np.abs((1 - b1) * coef * g), b2 * v + (1 - b2) * (coef * g) ** 2
    em, ev = 12 * U * m1, 16 * U * v1
    fix = 16 * U * (1 / (1 - b1 ** t) + 1 / (1 - b2 ** t))
    step = lr * (m1 / (1 - b1 ** t)) / np.sqrt(np.maximum(v1 / (1 - b2 ** t), 1e-300))
    return 4 * U * np.abs(p) + step * (40 * U + fix) + 1e-37, em + 1e-37, ev + 1e-37


@pytest.mark.parametrize("pack", ["aligned", "packed", "mixed"])
@pytest.mark.parametrize("name", list(LISTS))
def test_adam(rt, name, pack):
    """mixed: the four tensors of a parameter sit at different alignments."""
    sizes = LISTS[name]
    flats = [tensors(sizes, 3 + i, {"aligned": False, "packed": True, "mixed": i % 2 == 1}[pack], s) for i, s in enumerate((1.0, 0.1, 0.01, 0.01))]
    flats[3][0].abs_()
    (pf, p), (gf, g), (mf, m), (vf, v) = flats
    start = [[t.cpu().numpy().copy() for t in ts] for ts in (p, g, m, v)]
    coef = torch.tensor([0.37], device="cuda")
    adv = torch.tensor([4.0, 0.0, 0.0], device="cuda")
    rt.LaunchAdamList(p, g, m, v, adv, lr=1e-2, grad_scale=coef)
    rt.Check()
    b1, b2, lr, eps, c = (float(np.float32(q)) for q in (0.9, 0.999, 1e-2, 1e-8, 0.37))
    assert adv[0].item() == 5
    for k, n in enumerate(sizes):
        p0, g0, m0, v0 = (s[k].astype(np.float64) for s in start)
        want = ref.adam(p0, g0, m0, v0, 5, c, b1, b2, lr, eps)
        bounds = adam_bound(p0, g0, m0, v0, 5, c, lr, b1, b2)
        for got, w, b in zip((p[k], m[k], v[k]), want, bounds):
            assert np.all(np.abs(got.cpu().numpy() - w) <= b)
        assert np.array_equal(g[k].cpu().numpy(), start[1][k])


def test_adam_matches_the_flat_entry(rt):
    """Same arithmetic per element as tt_adam_step, weight decay of both kinds, several steps, without advancing too."""
    sizes = [100, 4096, 333, 9000]
    flat, _ = tensors(sizes, 9, True)
    n = flat.numel()
    for kw in (dict(coupledWd=0.1), dict(decoupledFactor=0.99), {}):
        state = [[flat * s for s in (1.0, 0.1)] + [torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda"), torch.zeros(3, device="cuda")] for _ in range(2)]
        spans, at = [], 0
        for k in sizes + [n - sum(sizes)]:
            spans.append((at, k))
            at += k
        for step in range(3):
            p, g, m, v, adv = state[0]
            rt.LaunchAdam(p, g, m, v, adv, n, lr=1e-2, advance=step != 1, **kw)
            lists = [[t[o:o + k] for o, k in spans] for t in state[1][:4]]
            rt.LaunchAdamList(*lists, state[1][4], lr=1e-2, advance=step != 1, **kw)
        rt.Check()
        # The two kernels may contract their products and sums differently.  The effective gradient g' keeps its sign and size
        # over the steps (|g'| <= 0.2 |start|), so m and v add terms of one sign: a step's two products and a sum leave m
        # and v within 4 U and 6 U of their largest terms, on each side, three times.  So the two m differ by at most 24 U max|g'|, the
        # two v by 36 U max g'^2, and m / sqrt(v), which is at most 1.1 here, by 2 (12 + 9 + 6) U of itself (errors of m, of
        # sqrt(v), and of the quotient, the root and the corrections' products); p adds that times lr and 4 U |p|, three times.
        g = 0.2 * float(flat.abs().max())
        bounds = [(3 * 1.1e-2 * 54 * U, 12 * U), (0.0, 0.0), (24 * U * g, 0.0), (36 * U * g * g, 0.0), (0.0, 0.0)]
        for a, b, (atol, rtol) in zip(*state, bounds):
            assert torch.allclose(a, b, rtol=rtol, atol=atol), kw
        assert state[1][4][0].item() == 2


def test_adam_optimizer_clips_on_the_way(rt):
    """ops.Adam.Step(max_norm) against clipping in place and stepping."""
    sizes = [70, 4000, 5]
    _, p1 = tensors(sizes, 20, False)
    _, g1 = tensors(sizes, 21, False)
    p2, g2 = [t.clone() for t in p1], [t.clone() for t in g1]
    one, two = ops.Adam(p1, lr=1e-2, weight_decay=0.01), ops.Adam(p2, lr=1e-2, weight_decay=0.01)
    for _ in range(3):
        na = one.Step(g1, max_norm=1.5)
        clipped = [g.clone() for g in g2]
        nb = ops.ClipGradNorm(clipped, 1.5)
        assert two.Step(clipped) is None
        assert na.item() == nb.item()
    for a, b, in zip(p1 + one.M.tensors + one.V.tensors, p2 + two.M.tensors + two.V.tensors):
        assert torch.equal(a, b)
    assert all(torch.equal(a, b) for a, b in zip(g1, g2))
    w = ops.Adam([torch.ones(4, device="cuda")], lr=0.1, weight_decay=0.5, decoupled=True)
    w.Step([torch.zeros(4, device="cuda")])
    assert torch.allclose(w.Params.tensors[0], torch.full((4,), 0.95, device="cuda"), rtol=4 * U)


def test_step_replays_from_a_graph(rt):
    sizes = LISTS["control net"]
    _, p1 = tensors(sizes, 30, False)
    _, g = tensors(sizes, 31, False)
    p2 = [t.clone() for t in p1]
    eager, graphed = ops.Adam(p1, lr=1e-2), ops.Adam(p2, lr=1e-2)
    gl = TensorList(g)
    for _ in range(4):
        eager.Step(gl, max_norm=1.0)
    graphed.Step(gl, max_norm=1.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        graphed.Step(gl, max_norm=1.0)
    for _ in range(3):
        graph.replay()
    rt.Check()
    assert graphed.Adv[0].item() == 4
    assert all(torch.equal(a, b) for a, b in zip(p1, p2))


def test_the_same_tensor_twice_in_a_norm(rt):
    """A tensor that stands in the list twice counts twice in the norm (scale=False: nothing is written)."""
    t = torch.full((5000,), 2.0, device="cuda")
    norm = torch.zeros(1, device="cuda")
    rt.LaunchClipGradNormList([t, t], 1.0, norm_out=norm, scale=False)
    assert abs(norm.item() - (2 * 5000 * 4) ** 0.5) <= 2 * U * norm.item()


def test_refusals(rt):
    import ctypes
    t = torch.ones(8, device="cuda")
    adv = torch.zeros(3, device="cuda")
    L, h = rt._L, rt._h
    ptr = (ctypes.c_void_p * 1)(t.data_ptr())
    off = (ctypes.c_void_p * 1)(t.data_ptr() + 2)
    null = (ctypes.c_void_p * 1)(None)
    n, minus, zero = ((ctypes.c_longlong * 1)(v) for v in (4, -1, 0))
    clip = lambda c, p, s: L.tt_clip_grad_norm_list(h, None, c, p, s, 1.0, 0.0, 1, None, None)      # noqa: E731
    assert clip(-1, ptr, n) == 1 and clip(1, None, n) == 1 and clip(1, ptr, None) == 1 and clip(1, null, n) == 1
    assert clip(1, ptr, minus) == 1 and clip(1, off, n) == 1 and clip((1 << 20) + 1, ptr, n) == 1
    assert clip(1, null, zero) == 0 and clip(0, None, None) == 0
    adam = lambda p, g, m, v, a: L.tt_adam_step_list(h, None, 1, p, g, m, v, n, a, None, 0.9, 0.99, 1e-3, 1e-8, 0.0, 1.0, 1)   # noqa: E731
    a = ctypes.c_void_p(adv.data_ptr())
    for bad in (0, 1, 2, 3):
        args = [ptr] * 4
        args[bad] = null
        assert adam(*args, a) == 1
    assert adam(ptr, ptr, ptr, ptr, None) == 1
    with pytest.raises(TensotronGemmError):
        rt.LaunchAdamList([t], [t[:4]], [t], [t], adv)
    with pytest.raises(TensotronGemmError):
        ops.Adam([t]).Step([t, t])
    with pytest.raises(TypeError):
        TensorList([t.double()])
    with pytest.raises(TypeError):
        TensorList([torch.ones((4, 4), device="cuda").t()[:, :2]])
    tiny = TensorRuntime(0, 4096)
    with pytest.raises(TensotronGemmError) as err:
        tiny.LaunchClipGradNormList([t], 1.0)
    assert err.value.status == 4
    tiny.Dispose()


FIRST_CALL = """
import torch
from tensotron_b200.runtime import LoraAdapters, TensorList, TensorRuntime
rt = TensorRuntime(0)
f = lambda *s: torch.ones(s, device="cuda")
lists = [TensorList([f(40000), f(3)]) for _ in range(4)]
adv, coef = torch.zeros(3, device="cuda"), torch.zeros(1, device="cuda")
ad = LoraAdapters(f(2, 4, 64), f(2, 48, 4))
rows = []
for m in (3, 100):
    idx = torch.arange(m, device="cuda", dtype=torch.int32) % 3 - 1
    rows.append((m, idx, f(m, 64), f(48, 64), f(m, 48), f(m, 4), f(m, 64), f(2, 4, 64), f(2, 48, 4), f(48, 64)))
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    rt.LaunchClipGradNormList(lists[1], 1.0, coef_out=coef, scale=False)
    rt.LaunchAdamList(*lists, adv, grad_scale=coef)
    rt.LaunchClipGradNormList(lists[1], 100.0)
    for m, idx, x, w, y, t, dx, da, db, dw in rows:
        rt.LaunchLoraForward(ad, idx, x, w, None, y, t, m, 48, 64)
        rt.LaunchLoraBackward(ad, idx, x, w, None, y, t, dx, None, None, da, db, m, 48, 64)
        rt.LaunchLoraBackward(ad, idx, x, w, None, y, t, dx, dw, None, da, db, m, 48, 64)
graph.replay()
rt.Check()
assert adv[0].item() == 1 and abs(coef.item() - 40003 ** -0.5) < 1e-6
for m, idx, x, w, y, t, *_ in rows:
    has = (idx >= 0).float()
    assert torch.equal(t, (64 * has)[:, None].expand(m, 4)) and torch.equal(y, (64 + 256 * has)[:, None].expand(m, 48))
print("captured first")
"""


def test_a_first_call_may_be_inside_a_capture(gemm_lib):
    import os
    import subprocess
    import sys
    from conftest import ROOT
    r = subprocess.run([sys.executable, "-c", FIRST_CALL], cwd=ROOT, env=dict(os.environ, PYTHONPATH=ROOT), capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured first" in r.stdout, r.stdout + r.stderr
