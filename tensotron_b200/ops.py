"""Host-side mirror of the reference's matmul op surface, on top of TensorRuntime.

Follows src/Tensotron/TensorOps.cs:211-279 (MatMul rank promotion, MatMul2D and its
stride-swap backward), src/Tensotron/TensorOps.MatMulND.cs:11-132 (batch broadcast,
RawBmm, batched backward, Bmm/Mv/Dot/Outer), src/Tensotron/TensorOps.LinearNT.cs:13-51
(MatMulNT) and src/Tensotron/Module.cs:82-112 (Linear).  Tensors are contiguous
float32 torch CUDA tensors used purely as device buffers; every product goes through
the C-ABI library.  Backward functions return the gradients the reference's GradNode
closures would hand to AddGrad.
"""
import math

import torch

from .runtime import ACT, Conv2dDesc, LoraAdapters, TensorList, TensorRuntime, TensotronGemmError, broadcast_batch

_runtime = {}


def runtime(device=None):
    """Process-wide runtime per device (TensorRuntime.Instance, src/Tensotron/TensorRuntime.cs:49-50)."""
    if device is None:
        device = torch.cuda.current_device()
    if device not in _runtime:
        _runtime[device] = TensorRuntime(device)
    return _runtime[device]


def _strides(shape):
    s, acc = [], 1
    for d in reversed(shape):
        s.append(acc)
        acc *= d
    return list(reversed(s))


def _check(t):
    if t.dtype != torch.float32 or not t.is_cuda or not t.is_contiguous():
        raise TensotronGemmError(1, "operands must be contiguous float32 CUDA tensors")


# ---- 2-D ---------------------------------------------------------------------------

def _matmul2d(a, b):
    M, K = a.shape
    K2, N = b.shape
    if K != K2:
        raise TensotronGemmError(1, "MatMul inner dims differ: %s @ %s." % (list(a.shape), list(b.shape)))
    out = torch.empty((M, N), dtype=torch.float32, device=a.device)
    runtime(a.device.index).LaunchMatMul(a, b, out, M, N, K, K, 1, N, 1)
    return out


def _matmul2d_backward(a, b, g):
    M, K = a.shape
    N = b.shape[1]
    rt = runtime(a.device.index)
    dA = torch.empty((M, K), dtype=torch.float32, device=a.device)
    rt.LaunchMatMul(g, b, dA, M, K, N, N, 1, 1, N)      # dA = g . B^T  (TensorOps.cs:264)
    dB = torch.empty((K, N), dtype=torch.float32, device=a.device)
    rt.LaunchMatMul(a, g, dB, K, N, M, 1, K, N, 1)      # dB = A^T . g  (TensorOps.cs:272)
    return dA, dB


# ---- N-D ---------------------------------------------------------------------------

def _raw_bmm(a, b, M, N, K, aMs, aKs, bKs, bNs, batch_dims, aBs, bBs):
    count = 1
    for d in batch_dims:
        count *= d
    out = torch.empty(tuple(batch_dims) + (M, N), dtype=torch.float32, device=a.device)
    runtime(a.device.index).LaunchMatMulBatched(a, b, out, count, M, N, K, aMs, aKs, bKs, bNs,
                                                batch_dims, aBs, bBs)
    return out


def _reduce_grad_to_shape(g, shape):
    """ReduceGradToShape (src/Tensotron/TensorOps.cs:76-100): sum over broadcast axes.  Only
    reached when the broadcast axes cannot be fused into the batched GEMM (they do not merge
    into one strided axis); then a fixed-order reduction kernel behind the C ABI does the sum."""
    shape = tuple(shape)
    if tuple(g.shape) == shape:
        return g.clone()
    r = g.dim()
    reduce_axis = []
    for j in range(r):
        axt = j - (r - len(shape))
        dt = shape[axt] if axt >= 0 else 1
        reduce_axis.append(1 if dt != g.shape[j] else 0)
    out = torch.empty(shape, dtype=torch.float32, device=g.device)
    runtime(g.device.index).LaunchReduceSumAxes(g, out, list(g.shape), reduce_axis)
    return out


def _bmm_reduced(x, y, M, N, K, xMs, xKs, yKs, yNs, batch_dims, xBs, yBs, target_shape):
    """RawBmm followed by ReduceGradToShape(., target_shape), fused into one launch when the
    broadcast axes merge into one (src/Tensotron/TensorOps.MatMulND.cs:80-103); otherwise the
    unfused pair."""
    r = len(batch_dims)
    tb = tuple(target_shape[:-2])
    reduce_axis = []
    for j in range(r):
        axt = j - (r - len(tb))
        dt = tb[axt] if axt >= 0 else 1
        reduce_axis.append(1 if dt != batch_dims[j] else 0)
    if any(reduce_axis):
        out = torch.empty(tuple(target_shape), dtype=torch.float32, device=x.device)
        try:
            runtime(x.device.index).LaunchMatMulBatchedReduce(x, y, out, M, N, K, xMs, xKs, yKs, yNs,
                                                              batch_dims, xBs, yBs, reduce_axis)
            return out
        except TensotronGemmError as e:
            if e.status != 3:
                raise
    full = _raw_bmm(x, y, M, N, K, xMs, xKs, yKs, yNs, batch_dims, xBs, yBs)
    return _reduce_grad_to_shape(full, target_shape)


def _matmul_nd(a, b):
    ar, br = a.dim(), b.dim()
    M, K = a.shape[-2], a.shape[-1]
    K2, N = b.shape[-2], b.shape[-1]
    if K != K2:
        raise TensotronGemmError(1, "MatMul inner dims differ: %s @ %s." % (list(a.shape), list(b.shape)))
    a_str, b_str = _strides(a.shape), _strides(b.shape)
    dims, aBs, bBs = broadcast_batch(a.shape[:-2], a_str[:-2], b.shape[:-2], b_str[:-2])
    return _raw_bmm(a, b, M, N, K, K, 1, N, 1, dims, aBs, bBs)


def _matmul_nd_backward(a, b, g):
    ar, br = a.dim(), b.dim()
    M, K = a.shape[-2], a.shape[-1]
    N = b.shape[-1]
    a_str, b_str, g_str = _strides(a.shape), _strides(b.shape), _strides(g.shape)
    gMs, gNs = g_str[-2], g_str[-1]
    # dA[.,m,k] = sum_n g[.,m,n] * B[.,k,n]   (TensorOps.MatMulND.cs:80-91)
    bd, gBs2, bBs2 = broadcast_batch(g.shape[:-2], g_str[:-2], b.shape[:-2], b_str[:-2])
    dA = _bmm_reduced(g, b, M, K, N, gMs, gNs, b_str[-1], b_str[-2], bd, gBs2, bBs2, a.shape)
    # dB[.,k,n] = sum_m A[.,m,k] * g[.,m,n]   (TensorOps.MatMulND.cs:92-103)
    bd, aBs2, gBs3 = broadcast_batch(a.shape[:-2], a_str[:-2], g.shape[:-2], g_str[:-2])
    dB = _bmm_reduced(a, g, K, N, M, a_str[-1], a_str[-2], gMs, gNs, bd, aBs2, gBs3, b.shape)
    return dA, dB


# ---- public surface -----------------------------------------------------------------

def MatMul(a, b):
    """TensorOps.MatMul (src/Tensotron/TensorOps.cs:211-240): torch matmul promotion rules."""
    _check(a), _check(b)
    if a.dim() == 2 and b.dim() == 2:
        return _matmul2d(a, b)
    if a.dim() == 1 and b.dim() == 2:
        return _matmul2d(a.reshape(1, -1), b).reshape(b.shape[1])
    if a.dim() == 2 and b.dim() == 1:
        return _matmul2d(a, b.reshape(-1, 1)).reshape(a.shape[0])
    if a.dim() == 1 and b.dim() == 1:
        return _matmul2d(a.reshape(1, -1), b.reshape(-1, 1)).reshape(())
    if a.dim() == 1:
        res = _matmul_nd(a.reshape(1, -1), b)
        return res.reshape(res.shape[:-2] + res.shape[-1:])
    if b.dim() == 1:
        res = _matmul_nd(a, b.reshape(-1, 1))
        return res.reshape(res.shape[:-1])
    return _matmul_nd(a, b)


def MatMulBackward(a, b, g):
    """The (dA, dB) the MatMul GradNode closures produce for upstream gradient g."""
    _check(a), _check(b), _check(g)
    if a.dim() == 2 and b.dim() == 2:
        return _matmul2d_backward(a, b, g)
    if a.dim() == 1 and b.dim() == 2:
        dA, dB = _matmul2d_backward(a.reshape(1, -1), b, g.reshape(1, -1))
        return dA.reshape(a.shape), dB
    if a.dim() == 2 and b.dim() == 1:
        dA, dB = _matmul2d_backward(a, b.reshape(-1, 1), g.reshape(-1, 1))
        return dA, dB.reshape(b.shape)
    if a.dim() == 1 and b.dim() == 1:
        dA, dB = _matmul2d_backward(a.reshape(1, -1), b.reshape(-1, 1), g.reshape(1, 1))
        return dA.reshape(a.shape), dB.reshape(b.shape)
    if a.dim() == 1:
        a2 = a.reshape(1, -1)
        g2 = g.reshape(g.shape[:-1] + (1, g.shape[-1]))
        dA, dB = _matmul_nd_backward(a2, b, g2.contiguous())
        return dA.reshape(a.shape), dB
    if b.dim() == 1:
        b2 = b.reshape(-1, 1)
        g2 = g.reshape(g.shape + (1,))
        dA, dB = _matmul_nd_backward(a, b2, g2.contiguous())
        return dA, dB.reshape(b.shape)
    return _matmul_nd_backward(a, b, g)


def Bmm(a, b):
    """TensorOps.Bmm (src/Tensotron/TensorOps.MatMulND.cs:110-118)."""
    if a.dim() != 3 or b.dim() != 3:
        raise TensotronGemmError(1, "bmm expects 3D tensors, got %s and %s." % (list(a.shape), list(b.shape)))
    if a.shape[0] != b.shape[0]:
        raise TensotronGemmError(1, "bmm batch sizes differ: %d vs %d." % (a.shape[0], b.shape[0]))
    _check(a), _check(b)
    return _matmul_nd(a, b)


def Mv(mat, vec):
    return MatMul(mat, vec)


def Dot(a, b):
    return MatMul(a, b)


def Outer(a, b):
    """TensorOps.Outer (src/Tensotron/TensorOps.MatMulND.cs:126-131)."""
    if a.dim() != 1 or b.dim() != 1:
        raise TensotronGemmError(1, "outer expects 1D tensors, got %s and %s." % (list(a.shape), list(b.shape)))
    return MatMul(a.reshape(-1, 1), b.reshape(1, -1))


def MatMulNT(a, b):
    """y = a . b^T without materialising b^T (src/Tensotron/TensorOps.LinearNT.cs:13-25)."""
    if a.dim() != 2 or b.dim() != 2:
        raise TensotronGemmError(1, "MatMulNT expects 2D operands, got %s and %s." % (list(a.shape), list(b.shape)))
    _check(a), _check(b)
    M, K = a.shape
    N, K2 = b.shape
    if K != K2:
        raise TensotronGemmError(1, "MatMulNT inner dims differ: %s . %s^T." % (list(a.shape), list(b.shape)))
    out = torch.empty((M, N), dtype=torch.float32, device=a.device)
    runtime(a.device.index).LaunchMatMul(a, b, out, M, N, K, K, 1, 1, K)
    return out


def MatMulNTBackward(a, b, g):
    """da = g . b (NN), db = g^T . a (TN) (src/Tensotron/TensorOps.LinearNT.cs:27-48)."""
    M, K = a.shape
    N = b.shape[0]
    rt = runtime(a.device.index)
    dA = torch.empty((M, K), dtype=torch.float32, device=a.device)
    rt.LaunchMatMul(g, b, dA, M, K, N, N, 1, K, 1)
    dB = torch.empty((N, K), dtype=torch.float32, device=a.device)
    rt.LaunchMatMul(g, a, dB, N, K, M, 1, N, K, 1)
    return dA, dB


def _conv_desc(x, weight, stride, padding, dilation):
    if x.dim() != 4:
        raise TensotronGemmError(1, "Conv2d expects (N,C,H,W), got %s." % list(x.shape))
    if weight.dim() != 4:
        raise TensotronGemmError(1, "Conv2d weight must be (O,C,kh,kw), got %s." % list(weight.shape))
    if weight.shape[1] != x.shape[1]:
        raise TensotronGemmError(1, "Conv2d channel mismatch: input %d vs weight %d." % (x.shape[1], weight.shape[1]))
    d = Conv2dDesc()
    d.n, d.c, d.h, d.w = (int(v) for v in x.shape)
    d.o, d.kh, d.kw = int(weight.shape[0]), int(weight.shape[2]), int(weight.shape[3])
    d.stride, d.padding, d.dilation = int(stride), int(padding), int(dilation)
    ho = (d.h + 2 * d.padding - d.dilation * (d.kh - 1) - 1) // d.stride + 1
    wo = (d.w + 2 * d.padding - d.dilation * (d.kw - 1) - 1) // d.stride + 1
    if ho <= 0 or wo <= 0:
        raise TensotronGemmError(1, "Im2Col: non-positive output size (%dx%d) for %s." % (ho, wo, list(x.shape)))
    return d, ho, wo


def Conv2d(x, weight, bias=None, stride=1, padding=0, dilation=1):
    """TensorOps.Conv2d (src/Tensotron/TensorOps.Conv.cs:60-80): im2col + batched matmul + bias, on
    the batched GEMM engine.  The handle workspace must hold the columns
    (TensorRuntime.Conv2dWorkspace)."""
    _check(x), _check(weight)
    d, ho, wo = _conv_desc(x, weight, stride, padding, dilation)
    y = torch.empty((d.n, d.o, ho, wo), dtype=torch.float32, device=x.device)
    runtime(x.device.index).LaunchConv2dForward(d, x, weight, bias, y)
    return y


def Conv2dBackward(x, weight, g, stride=1, padding=0, dilation=1, need_dx=True, has_bias=True):
    """(dx, dW, dbias) for upstream gradient g of Conv2d's output: what the reference's autograd
    chain (bias add, broadcast matmul, Im2Col) hands to AddGrad."""
    _check(x), _check(weight), _check(g)
    d, _, _ = _conv_desc(x, weight, stride, padding, dilation)
    dx = torch.empty_like(x) if need_dx else None
    dw = torch.empty_like(weight)
    db = torch.empty((d.o,), dtype=torch.float32, device=x.device) if has_bias else None
    runtime(x.device.index).LaunchConv2dBackward(d, x, weight, g, dx, dw, db)
    return dx, dw, db


class Linear:
    """y = act(x . W^T + b): Linear (src/Tensotron/Module.cs:82-112) with the Activation
    module that follows it fused into the GEMM epilogue.  Weight is (out, in)."""

    def __init__(self, in_features, out_features, bias=True, act=None, device="cuda", generator=None):
        bound = 1.0 / math.sqrt(in_features)  # Kaiming-uniform a=sqrt(5) (src/Tensotron/Init.cs:54-58)
        self.Weight = (torch.rand((out_features, in_features), generator=generator) * 2 - 1).mul_(bound).to(device)
        self.Bias = ((torch.rand((out_features,), generator=generator) * 2 - 1).mul_(bound).to(device)
                     if bias else None)
        self.act = ACT[act]

    def Forward(self, x):
        _check(x)
        M, K = x.shape
        N = self.Weight.shape[0]
        y = torch.empty((M, N), dtype=torch.float32, device=x.device)
        runtime(x.device.index).LaunchLinearForward(x, self.Weight, self.Bias, y, M, N, K, self.act)
        return y

    def Backward(self, x, y, dy, need_dx=True):
        """Returns (dx, dW, dbias) for upstream gradient dy of the activated output y."""
        M, K = x.shape
        N = self.Weight.shape[0]
        dx = torch.empty((M, K), dtype=torch.float32, device=x.device) if need_dx else None
        dw = torch.empty((N, K), dtype=torch.float32, device=x.device)
        db = torch.empty((N,), dtype=torch.float32, device=x.device) if self.Bias is not None else None
        runtime(x.device.index).LaunchLinearBackward(x, self.Weight, y, dy, dx, dw, db, M, N, K, self.act)
        return dx, dw, db


class LoraLinear(Linear):
    """A Linear whose rows bring their own low-rank adapters (no counterpart in the reference): `adapters` pairs
    A (rank, in), B (out, rank) beside the one projection, y = act(x . W^T + b + Scale[e] * (x . A[e]^T) . B[e]^T) for a
    row with adapter e.  A starts like a Linear's weight, B at zero, Scale at alpha / rank."""

    def __init__(self, in_features, out_features, rank, adapters=1, alpha=None, bias=True, act=None, device="cuda", generator=None):
        super().__init__(in_features, out_features, bias=bias, act=act, device=device, generator=generator)
        bound = 1.0 / math.sqrt(in_features)
        self.A = (torch.rand((adapters, rank, in_features), generator=generator) * 2 - 1).mul_(bound).to(device)
        self.B = torch.zeros((adapters, out_features, rank), device=device)
        self.Scale = torch.full((adapters,), (rank if alpha is None else alpha) / rank, device=device)

    def _adapters(self):
        # (made again when a tensor was replaced: the description holds addresses)
        d = getattr(self, "_desc", None)
        if d is None or d.a is not self.A or d.b is not self.B or d.scale is not self.Scale:
            d = self._desc = LoraAdapters(self.A, self.B, self.Scale)
        return d

    def _check_rows(self, x, row_adapter):
        _check(x)
        n, k = self.Weight.shape
        if x.dim() != 2 or x.shape[1] != k:
            raise TensotronGemmError(1, "LoraLinear expects (rows, %d), got %s." % (k, list(x.shape)))
        if self.A.shape[2] != k or self.B.shape[1] != n:
            raise TensotronGemmError(1, "adapters of another layer: A %s, B %s, W %s." % (list(self.A.shape), list(self.B.shape), [n, k]))
        if row_adapter is not None and (row_adapter.dtype != torch.int32 or not row_adapter.is_contiguous() or
                                        row_adapter.device != x.device or tuple(row_adapter.shape) != (x.shape[0],)):
            raise TensotronGemmError(1, "row_adapter must be %d int32 values on the rows' device." % x.shape[0])
        return x.shape[0], n, k

    def Forward(self, x, row_adapter=None):
        """Returns (y, t): the output and the down-projected rows that Backward takes.  row_adapter: int32 (rows), -1 for a
        row without an adapter; None: adapter 0 for every row."""
        M, N, K = self._check_rows(x, row_adapter)
        y = torch.empty((M, N), dtype=torch.float32, device=x.device)
        t = torch.empty((M, self.A.shape[1]), dtype=torch.float32, device=x.device)
        runtime(x.device.index).LaunchLoraForward(self._adapters(), row_adapter, x, self.Weight, self.Bias, y, t, M, N, K, self.act)
        return y, t

    def Backward(self, x, y, t, dy, row_adapter=None, need_dx=True, need_base=False):
        """Returns (dx, dA, dB, dW, dbias); dW and dbias only with need_base (a frozen projection has none).  t None:
        recomputed from x."""
        M, N, K = self._check_rows(x, row_adapter)
        for v, shape in ((y, (M, N)), (dy, (M, N)), (t, (M, self.A.shape[1]))):
            if v is not None:
                _check(v)
                if tuple(v.shape) != shape:
                    raise TensotronGemmError(1, "LoraLinear.Backward expects %s, got %s." % (list(shape), list(v.shape)))
        new = lambda want, like: torch.empty_like(like) if want and like is not None else None   # noqa: E731
        dx, da, db = new(need_dx, x), torch.empty_like(self.A), torch.empty_like(self.B)
        dw, dbias = new(need_base, self.Weight), new(need_base, self.Bias)
        runtime(x.device.index).LaunchLoraBackward(self._adapters(), row_adapter, x, self.Weight, y, dy, t, dx, dw, dbias, da, db,
                                                   M, N, K, self.act)
        return dx, da, db, dw, dbias


def ClipGradNorm(grads, max_norm, eps=1e-6):
    """GradUtils.ClipGradNorm (src/Tensotron/Optimizers.cs:383-422) over a list of gradients: scales all of them in place
    by clamp(max_norm / (norm + eps), 0, 1) and returns the norm before it (device scalar)."""
    grads = grads if isinstance(grads, TensorList) else TensorList(grads)
    device = torch.cuda.current_device() if grads.device is None else grads.device
    norm = torch.empty(1, dtype=torch.float32, device=torch.device("cuda", device))
    runtime(device).LaunchClipGradNormList(grads, max_norm, eps, norm_out=norm)
    return norm


class Adam:
    """Adam / AdamW over a parameter list (src/Tensotron/Optimizers.cs:144-233), one launch per step, the step counter on
    the device.  weight_decay is coupled (added to the gradient) unless decoupled."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, decoupled=False):
        self.Params = TensorList(params)
        if not self.Params.count:
            raise ValueError("Adam needs at least one parameter")
        self.lr, self.betas, self.eps, self.weight_decay, self.decoupled = lr, betas, eps, weight_decay, decoupled
        self.M = TensorList([torch.zeros_like(p) for p in self.Params.tensors])
        self.V = TensorList([torch.zeros_like(p) for p in self.Params.tensors])
        dev = self.Params.tensors[0].device
        self.Adv = torch.zeros(3, device=dev)
        self._norm, self._coef = torch.zeros(1, device=dev), torch.zeros(1, device=dev)

    def Step(self, grads, max_norm=None, clip_eps=1e-6):
        """One step.  max_norm: the gradients' global norm is clipped to it on the way (the tensors in `grads` stay as
        they are); returns that norm (device scalar), else None."""
        grads = grads if isinstance(grads, TensorList) else TensorList(grads)
        if grads.numels != self.Params.numels:
            raise TensotronGemmError(1, "gradients differ from the parameters in number or sizes")
        rt = runtime(self.Params.device)
        if max_norm is not None:
            rt.LaunchClipGradNormList(grads, max_norm, clip_eps, norm_out=self._norm, coef_out=self._coef, scale=False)
        coupled = 0.0 if self.decoupled else self.weight_decay
        factor = 1.0 - self.lr * self.weight_decay if self.decoupled else 1.0
        rt.LaunchAdamList(self.Params, grads, self.M, self.V, self.Adv, b1=self.betas[0], b2=self.betas[1], lr=self.lr, eps=self.eps,
                          coupledWd=coupled, decoupledFactor=factor, grad_scale=self._coef if max_norm is not None else None)
        return self._norm if max_norm is not None else None
