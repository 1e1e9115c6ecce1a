"""CPU suite of the adapter and list operators: the 64-bit restatement's gradients against differences, the host-side
checks, and the status codes that need no device."""
import ctypes

import numpy as np
import pytest
import torch

import adapters_ref as ref
from tensotron_b200 import ops, runtime


@pytest.mark.parametrize("kind,mix", [("none", "mixed"), ("tanh", "sorted"), ("relu", "one"), ("none", "none")])
def test_restated_gradients_against_differences(kind, mix):
    m, n, k, r, e = 7, 5, 6, 3, 3
    d = {name: v if v is None or name == "idx" else v.astype(np.float64) for name, v in ref.inputs(3, m, n, k, r, e, mix).items()}
    y, t, _, _ = ref.forward(d["x"], d["w"], d["bias"], d["a"], d["b"], d["s"], d["idx"], kind)
    got = ref.backward(d["x"], d["w"], d["a"], d["b"], d["s"], d["idx"], kind, y, d["dy"], t)

    def loss(**change):
        q = {**d, **change}
        return float((ref.forward(q["x"], q["w"], q["bias"], q["a"], q["b"], q["s"], q["idx"], kind)[0] * d["dy"]).sum())

    h = 1e-6
    for name, grad in (("x", "dx"), ("a", "da"), ("b", "db"), ("w", "dw"), ("bias", "dbias")):
        num = np.zeros_like(d[name])
        for at in np.ndindex(*d[name].shape):
            up, down = d[name].copy(), d[name].copy()
            up[at] += h
            down[at] -= h
            num[at] = (loss(**{name: up}) - loss(**{name: down})) / (2 * h)
        # central differences: curvature h^2 and rounding 1e-16 / h, both far below 1e-6
        np.testing.assert_allclose(got[grad][0], num, atol=1e-6, rtol=1e-6)


def test_entries_without_a_handle_return_status_codes(gemm_lib):
    assert gemm_lib.tt_lora_fwd(None, None, None, None, None, None, None, None, None, 1, 1, 1, 0) == 1
    assert gemm_lib.tt_lora_bwd(None, None, None, *[None] * 11, 1, 1, 1, 0) == 1
    assert gemm_lib.tt_clip_grad_norm_list(None, None, 0, None, None, 1.0, 0.0, 1, None, None) == 1
    assert gemm_lib.tt_adam_step_list(None, None, 0, *[None] * 4, None, None, None, 0.9, 0.99, 1e-3, 1e-8, 0.0, 1.0, 1) == 1


def test_workspace_query(gemm_lib):
    f = runtime.TensorRuntime.LoraWorkspace
    assert f(-1, 4, 4, 1, 1) == 0 and f(4, 4, 4, 0, 1) == 0
    small, large = f(64, 64, 128, 4, 8), f(8192, 64, 128, 4, 8)
    assert 4 * 64 * 9 <= small < large
    # a backward call keeps dt, and with an activation the masked gradient
    assert f(64, 64, 128, 4, 8, backward=True) >= small + 4 * 64 * 8
    assert f(64, 64, 128, 4, 8, act="relu", backward=True) >= f(64, 64, 128, 4, 8, backward=True) + 4 * 64 * 64


def test_host_objects_refuse_what_the_kernels_cannot_read():
    cpu = torch.zeros(2, 3, 4)
    with pytest.raises(TypeError):
        runtime.LoraAdapters(cpu, torch.zeros(2, 5, 3))
    with pytest.raises(TypeError):
        runtime.TensorList([torch.zeros(3)])
    assert runtime.TensorList([]).count == 0
    assert ctypes.sizeof(runtime.LoraDesc) == 32
    with pytest.raises(ValueError):
        ops.Adam([])
