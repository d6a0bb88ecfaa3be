"""Device-tensor entry points over the C ABI (the ``*_dev`` functions).

torch is plumbing here: it owns device memory and the stream.  Every call
launches the gfx950 kernels of libkatsu_hip.so on torch's current stream;
nothing is computed by torch.  Host (numpy) entry points live in
``katsu_amd.host``.
"""
import ctypes
from array import array

import torch

from ._abi import (BF16, F32, Attention, AttentionGrads, BlockNorm, Distillation, Embedding,
                   QkNormRotary, QkNormRotaryGrads, Rotary, check, geometry, lib)


# A small call's time is its host side (a pass of four 48 x 56 products and
# fills took 31 us, the GPU 14): the stream as the raw handle torch's own
# launchers read (0.3 us, against 2.9 through torch.cuda.current_stream()'s
# Stream object), pointers as integers, which the argtypes convert.  The names
# are looked up per call: a torch without a GPU build does not have them.
def _stream():
    c = torch._C
    return c._cuda_getCurrentRawStream(c._cuda_getDevice())


def _p(t):
    return t.data_ptr() if t is not None and t.numel() else 0


def _dev_f32(*ts):
    for t in ts:
        if t is not None and not (t.is_cuda and t.dtype is torch.float32 and t.is_contiguous()):
            raise ValueError("katsu_amd.ops expects contiguous float32 device tensors")


def conv_geom(xshape, wshape, stride, pad):
    n, c, h, w = xshape
    k, c2, r, s = wshape
    if c != c2:
        raise ValueError("input channels must match weights")
    return geometry(n, c, h, w, k, r, s, stride, pad)


def conv2d_forward(x, w, stride, pad, out=None):
    """y = conv(x, w): Conv2D::forward (conv2d.rs:95-115)."""
    _dev_f32(x, w, out)
    g = conv_geom(x.shape, w.shape, stride, pad)
    if out is None:
        out = torch.empty((g.n, g.k, g.oh, g.ow), device=x.device, dtype=torch.float32)
    check(lib().katsu_hip_conv2d_fwd_f32_dev(_p(x), _p(w), _p(out), ctypes.byref(g), _stream()),
          "conv2d_fwd")
    return out


def conv2d_backward_data(gy, w, xshape, stride, pad, out=None, beta=0.0):
    """dx (conv2d.rs:288); beta=1 accumulates into `out`."""
    _dev_f32(gy, w, out)
    g = conv_geom(xshape, w.shape, stride, pad)
    if out is None:
        out = torch.empty(tuple(xshape), device=gy.device, dtype=torch.float32)
    check(lib().katsu_hip_conv2d_bwd_data_f32_dev(_p(gy), _p(w), _p(out), ctypes.byref(g),
                                                   float(beta), _stream()), "conv2d_bwd_data")
    return out


def bwd_filter_workspace_bytes(xshape, wshape, stride, pad):
    g = conv_geom(xshape, wshape, stride, pad)
    nbytes = ctypes.c_size_t(0)
    check(lib().katsu_hip_conv2d_bwd_filter_workspace(ctypes.byref(g), ctypes.byref(nbytes)),
          "bwd_filter_workspace")
    return nbytes.value


def conv2d_backward_filter(x, gy, wshape, stride, pad, out=None, beta=0.0, workspace=None):
    """dw (conv2d.rs:289); beta=1 accumulates into `out`.

    `workspace` is an optional uint8/float device tensor of at least
    bwd_filter_workspace_bytes(); without it the library's own buffer is used."""
    _dev_f32(x, gy, out)
    g = conv_geom(x.shape, wshape, stride, pad)
    if out is None:
        out = torch.empty(tuple(wshape), device=x.device, dtype=torch.float32)
    ws = workspace.data_ptr() if workspace is not None else 0
    wsb = workspace.numel() * workspace.element_size() if workspace is not None else 0
    check(lib().katsu_hip_conv2d_bwd_filter_f32_dev(_p(x), _p(gy), _p(out), ctypes.byref(g),
                                                     float(beta), ws, wsb, _stream()),
          "conv2d_bwd_filter")
    return out


def conv2d_backward(x, w, gy, stride, pad, dx=None, dw=None, beta=0.0, workspace=None):
    """(dx, dw) of backward_buffers (conv2d.rs:265-292) in one call; beta=1
    accumulates into `dx` and `dw`.  When both passes take the direct gfx950
    kernels they run as a single launch.  `workspace` as for
    conv2d_backward_filter."""
    _dev_f32(x, w, gy, dx, dw)
    g = conv_geom(x.shape, w.shape, stride, pad)
    if dx is None:
        dx = torch.empty(tuple(x.shape), device=x.device, dtype=torch.float32)
    if dw is None:
        dw = torch.empty(tuple(w.shape), device=x.device, dtype=torch.float32)
    ws = workspace.data_ptr() if workspace is not None else 0
    wsb = workspace.numel() * workspace.element_size() if workspace is not None else 0
    check(lib().katsu_hip_conv2d_bwd_f32_dev(_p(x), _p(w), _p(gy), _p(dx), _p(dw),
                                              ctypes.byref(g), float(beta), ws, wsb, _stream()),
          "conv2d_bwd")
    return dx, dw


def gemm(a, b, m, n, k, trans_a=False, trans_b=False, out=None, beta=0.0):
    """out[m,n] = beta*out + op(a) op(b) (tensor.rs:264-273, 424-444)."""
    _dev_f32(a, b, out)
    if out is None:
        out = torch.empty((m, n), device=a.device, dtype=torch.float32)
    check(lib().katsu_hip_gemm_f32_dev(_p(a), _p(b), _p(out), m, n, k, int(trans_a),
                                       int(trans_b), float(beta), _stream()), "gemm")
    return out


def matmul(a, b):
    """Tensor::matmul forward: [m,k] @ [k,n] (tensor.rs:249-280)."""
    m, k = a.shape
    k2, n = b.shape
    if k != k2:
        raise ValueError("matmul inner dimensions differ")
    return gemm(a, b, m, n, k)


def matmul_vjp(a, b, g, da, db):
    """Matmul VJP (tensor.rs:418-445): da += g b^T, then db += a^T g.

    One call of katsu_hip_matmul_vjp_f32_dev: the two products run as one
    launch when da and db are separate buffers, and in the reference's order
    when they are the same tensor (A and B the same node)."""
    m, k = a.shape
    n = b.shape[1]
    if m * n == 0 or k == 0:
        return da, db
    _dev_f32(a, b, g, da, db)
    check(lib().katsu_hip_matmul_vjp_f32_dev(_p(a), _p(b), _p(g), _p(da), _p(db), m, k, n,
                                             1.0, 1.0, _stream()), "matmul_vjp")
    return da, db


# ---- the device engine's elementwise work (f32, n elements, device tensors) ----

def add(a, b, out=None, beta=0.0):
    """out = beta*out + (a + b): Tensor::add (tensor.rs:217-240), bit-exact."""
    _dev_f32(a, b, out)
    if a.shape != b.shape:
        raise ValueError("identical shapes required")
    out = torch.empty_like(a) if out is None else out
    check(lib().katsu_hip_add_f32_dev(_p(a), _p(b), _p(out), a.numel(), float(beta), _stream()),
          "add")
    return out


def mul(a, b, out=None, beta=0.0):
    """out = beta*out + a*b: Tensor::mul, or Mul's VJP with beta = 1."""
    _dev_f32(a, b, out)
    if a.shape != b.shape:
        raise ValueError("identical shapes required")
    out = torch.empty_like(a) if out is None else out
    check(lib().katsu_hip_mul_f32_dev(_p(a), _p(b), _p(out), a.numel(), float(beta), _stream()),
          "mul")
    return out


def accumulate(x, y, beta=1.0):
    """y = beta*y + x (an adjoint into a pending buffer)."""
    _dev_f32(x, y)
    check(lib().katsu_hip_accumulate_f32_dev(_p(x), _p(y), x.numel(), float(beta), _stream()),
          "accumulate")
    return y


def fill(x, value):
    _dev_f32(x)
    check(lib().katsu_hip_fill_f32_dev(_p(x), x.numel(), float(value), _stream()), "fill")
    return x


def add_scalar(s, y, beta=1.0):
    """y = beta*y + s[0] (Sum's VJP)."""
    _dev_f32(s, y)
    check(lib().katsu_hip_add_scalar_f32_dev(_p(s), _p(y), y.numel(), float(beta), _stream()),
          "add_scalar")
    return y


def sum(x, out=None, beta=0.0):
    """out[0] = beta*out[0] + sum(x): Tensor::sum (tensor.rs:242-247), fixed tree."""
    _dev_f32(x, out)
    out = torch.empty(1, device=x.device, dtype=torch.float32) if out is None else out
    check(lib().katsu_hip_sum_f32_dev(_p(x), x.numel(), _p(out), float(beta), _stream()), "sum")
    return out


def mean_rows(y, rows, cols, out=None):
    """out[r] = sum_c y[r][c] / cols (the stem chain's global average pool)."""
    _dev_f32(y, out)
    out = torch.empty(rows, device=y.device, dtype=torch.float32) if out is None else out
    check(lib().katsu_hip_mean_rows_f32_dev(_p(y), rows, cols, _p(out), _stream()), "mean_rows")
    return out


def broadcast_rows(g, rows, cols, scale, dy=None, beta=0.0):
    """dy[r][c] = beta*dy[r][c] + scale*g[r] (the mean pool's VJP)."""
    _dev_f32(g, dy)
    dy = torch.empty(rows * cols, device=g.device, dtype=torch.float32) if dy is None else dy
    check(lib().katsu_hip_broadcast_rows_f32_dev(_p(g), rows, cols, float(scale), _p(dy),
                                                  float(beta), _stream()), "broadcast_rows")
    return dy


def grad_cam(act, grad, size=None):
    """Grad-CAM of an NCHW activation map and its gradient: [N, H, W] maps,
    ReLU of the channel sum weighted by the gradient's spatial means, each
    divided by its maximum; with size=(OH, OW), each map then resized to the
    original image by resize_bilinear."""
    _dev_f32(act, grad)
    if act.shape != grad.shape or act.dim() != 4:
        raise ValueError("activation and gradient must be the same NCHW shape")
    n, c, h, w = act.shape
    cam = torch.empty((n, h, w), device=act.device, dtype=torch.float32)
    check(lib().katsu_hip_gradcam_f32_dev(_p(act), _p(grad), n, c, h * w, _p(cam), _stream()),
          "grad_cam")
    return cam if size is None else resize_bilinear(cam, size)


def resize_bilinear(maps, size):
    """[N, H, W] maps resized to [N, OH, OW]: bilinear, half-pixel centres."""
    _dev_f32(maps)
    if maps.dim() != 3:
        raise ValueError("maps must be [N, H, W]")
    n, h, w = maps.shape
    oh, ow = (int(v) for v in size)
    out = torch.empty((n, oh, ow), device=maps.device, dtype=torch.float32)
    check(lib().katsu_hip_resize_bilinear_f32_dev(_p(maps), n, h, w, oh, ow, _p(out),
                                                   _stream()), "resize_bilinear")
    return out


# ---- language-model operators (float32 or bfloat16 device tensors) ----

_DTYPE = {torch.float32: F32, torch.bfloat16: BF16}


def _dev_lm(first, *ts):
    """float32 or bfloat16 device tensors, all of the first one's type and device."""
    if not first.is_cuda or first.dtype not in _DTYPE:
        raise ValueError("float32 or bfloat16 device tensors expected")
    for t in ts:
        if t is not None and (t.dtype is not first.dtype or t.device != first.device):
            raise ValueError("all operands must have one type and device")


def _heads(t, what):
    """A [tokens, heads, channels] tensor's strides; its channels must be adjacent."""
    s = t.stride()
    if len(s) != 3 or (s[2] != 1 and t.shape[2] > 1):
        raise ValueError(f"{what} must be [tokens, heads, channels] with adjacent channels")
    return s[:2]


def _int32(t, n, dev, what):
    if t is not None and not (t.dtype is torch.int32 and t.device == dev and t.dim() == 1
                              and t.is_contiguous() and t.numel() == n):
        raise ValueError(f"{what} must be {n} contiguous int32 values on the operands' device")


def _attention(q, k, v, out, cu_q, cu_k, k_lens, causal, scale):
    _dev_lm(q, k, v, out)
    strides = [_heads(t, w) for t, w in ((q, "q"), (k, "k"), (v, "v"), (out, "out"))]
    tq, heads, dim = q.shape
    if k.shape != v.shape or k.shape[2] != dim or dim == 0 or out.shape != q.shape:
        raise ValueError("k and v must have one shape, q's channels (one at least), out q's shape")
    if k.shape[1] == 0 or heads % k.shape[1]:
        raise ValueError("query heads must be a multiple of key heads")
    if (cu_q is None) != (cu_k is None):
        raise ValueError("cu_q and cu_k go together")
    seqs = 1 if cu_q is None else cu_q.numel() - 1
    if seqs < 0:
        raise ValueError("cu_q holds the sequences' starts and the end")
    _int32(cu_q, seqs + 1, q.device, "cu_q")
    _int32(cu_k, seqs + 1, q.device, "cu_k")
    _int32(k_lens, seqs, q.device, "k_lens")
    return Attention(_DTYPE[q.dtype], bool(causal), heads, k.shape[1], dim, seqs, tq, k.shape[0],
                     *strides, dim ** -0.5 if scale is None else scale)


def attention_workspace_bytes(q, k, v, cu_q=None, cu_k=None, backward=False):
    """Scratch that attention (or attention_backward) needs for these operands."""
    d = _attention(q, k, v, q, cu_q, cu_k, None, True, None)
    nbytes = ctypes.c_size_t(0)
    fn = (lib().katsu_hip_attention_bwd_workspace if backward
          else lib().katsu_hip_attention_fwd_workspace)
    check(fn(ctypes.byref(d), ctypes.byref(nbytes)), "attention_workspace")
    return nbytes.value


def _workspace(t, dev):
    """A workspace's address and bytes: the kernels write it, so it must be memory of theirs."""
    if t is None:
        return 0, 0
    if t.device != dev or not t.is_contiguous():
        raise ValueError("workspace must be contiguous and on the operands' device")
    return t.data_ptr(), t.numel() * t.element_size()


def attention(q, k, v, cu_q=None, cu_k=None, k_lens=None, causal=True, scale=None, out=None,
              workspace=None):
    """(out, lse) of softmax(scale q k^T) v over packed sequences: q [Tq, H, D], k and v
    [Tk, Hkv, D], channels adjacent, any token and head strides; cu_q and cu_k the int32 starts
    of the sequences' queries and keys and the end (None: one sequence; a slice of a batch's starts
    gives those sequences); k_lens how many of each sequence's keys are in use (a cache's slots).
    causal: the last query sees every key, each earlier one a key less.  A query that sees no key
    gives 0 and lse -inf; the output of a token that no sequence holds is undefined, its gradients
    too.  scale: 1/sqrt(D) if None.  lse [H, Tq], float32, is what attention_backward takes.
    `workspace`: an optional device tensor of attention_workspace_bytes(); without it the library's
    own buffer is used."""
    out = torch.empty_like(q) if out is None else out
    d = _attention(q, k, v, out, cu_q, cu_k, k_lens, causal, scale)
    lse = torch.empty((q.shape[1], q.shape[0]), device=q.device, dtype=torch.float32)
    check(lib().katsu_hip_attention_fwd_dev(ctypes.byref(d), _p(q), _p(k), _p(v), _p(cu_q),
                                            _p(cu_k), _p(k_lens), _p(out), _p(lse),
                                            *_workspace(workspace, q.device), _stream()),
          "attention")
    return out, lse


def attention_backward(dout, q, k, v, out, lse, cu_q=None, cu_k=None, causal=True, scale=None,
                       dq=None, dk=None, dv=None, workspace=None):
    """(dq, dk, dv) of attention's out with gradient dout, from the forward call's operands and
    its out and lse.  Any token and head strides; `workspace` of
    attention_workspace_bytes(..., backward=True)."""
    d = _attention(q, k, v, out, cu_q, cu_k, None, causal, scale)
    dq = torch.empty_like(q) if dq is None else dq
    dk = torch.empty_like(k) if dk is None else dk
    dv = torch.empty_like(v) if dv is None else dv
    _dev_lm(q, dout, dq, dk, dv)
    if dout.shape != q.shape or dq.shape != q.shape or dk.shape != k.shape or dv.shape != k.shape:
        raise ValueError("gradients must have their operands' shapes")
    if (lse.dtype is not torch.float32 or lse.device != q.device or not lse.is_contiguous()
            or lse.shape != (q.shape[1], q.shape[0])):
        raise ValueError("lse must be what attention returned")
    g = AttentionGrads(*(_heads(t, w) for t, w in ((dout, "dout"), (dq, "dq"), (dk, "dk"),
                                                   (dv, "dv"))))
    check(lib().katsu_hip_attention_bwd_dev(ctypes.byref(d), ctypes.byref(g), _p(dout), _p(q),
                                            _p(k), _p(v), _p(out), _p(lse), _p(cu_q), _p(cu_k),
                                            _p(dq), _p(dk), _p(dv),
                                            *_workspace(workspace, q.device), _stream()),
          "attention_backward")
    return dq, dk, dv


def rotary_table(length, dim, base=10000.0, factor=1.0, by_wavelength=True, device="cuda"):
    """[length, dim] float32: the cosines and sines of `length` positions' angles for `dim`
    turning channels, computed in float64.  factor > 1: for a context of `length` tokens, factor
    times what the model was trained on: all frequencies divided by it, or (by_wavelength) only
    those that turn seldom within the original length."""
    t = torch.empty((length, dim), device=device, dtype=torch.float32)
    with torch.cuda.device(t.device):
        check(lib().katsu_hip_rotary_table_f32_dev(_p(t), length, dim, base, factor,
                                                   int(by_wavelength and factor != 1.0),
                                                   _stream()), "rotary_table")
    return t


def rotary(q, k, table, positions=None, interleaved=False, inverse=False, out_q=None, out_k=None):
    """(q', k'): the first table.shape[1] channels of each head of q and k [tokens, heads,
    channels] (k may be None) turned by their tokens' positions, rows of `table` (int32; None:
    0, 1, ..).  Pairs are channels i and i + R/2, or neighbours with interleaved.  inverse turns
    back: the gradient of a turn.  The outputs may be the inputs."""
    out_q = torch.empty_like(q) if out_q is None else out_q
    if k is not None and out_k is None:
        out_k = torch.empty_like(k)
    _dev_lm(q, k, out_q, out_k)
    tokens, heads, dim = q.shape if q.dim() == 3 else (0, 0, 0)
    strides = [(0, 0) if t is None else _heads(t, w)
               for t, w in ((q, "q"), (k, "k"), (out_q, "out_q"), (out_k, "out_k"))]
    if out_q.shape != q.shape or (k is not None and (
            out_k.shape != k.shape or k.shape[0] != tokens or k.shape[2] != dim)):
        raise ValueError("q and k must have the same tokens and channels, outputs their shapes")
    if (table.dim() != 2 or table.dtype is not torch.float32 or table.device != q.device
            or not table.is_contiguous()):
        raise ValueError("table must be contiguous float32 [length, channels that turn]")
    _int32(positions, tokens, q.device, "positions")
    d = Rotary(_DTYPE[q.dtype], bool(interleaved), bool(inverse), tokens, heads,
               0 if k is None else k.shape[1], dim, table.shape[1], table.shape[0], *strides)
    check(lib().katsu_hip_rotary_dev(ctypes.byref(d), _p(q), _p(k), _p(table), _p(positions),
                                     _p(out_q), _p(out_k), _stream()), "rotary")
    return out_q, out_k


def _block_norm(rows, gate, w_post, w_pre, alpha, eps):
    """Checks the operands of a block norm against its first [rows, cols] one."""
    first = rows[0]
    _dev_lm(*rows, gate, w_post, w_pre)
    if first.dim() != 2:
        raise ValueError("operands must be [rows, cols]")
    cols = first.shape[1]
    for t in rows:
        if t is not None and (t.shape != first.shape or not t.is_contiguous()):
            raise ValueError("operands must be contiguous and of one shape")
    for t in (w_post, w_pre):
        if t is not None and (t.shape != (cols,) or not t.is_contiguous()):
            raise ValueError("weights must be contiguous [cols]")
    if gate is not None and (gate.shape not in (first.shape, (cols,)) or not gate.is_contiguous()):
        raise ValueError("gate must be contiguous, [cols] or [rows, cols]")
    return BlockNorm(_DTYPE[first.dtype], 0 if gate is None else gate.dim(), *first.shape,
                     alpha, eps)


def block_norm(x, o, gate=None, w_post=None, w_pre=None, alpha=1.0, eps=1e-6, out_y=None,
               out_h=None):
    """(y, h, stats) between two blocks: o, a block's output, is divided by its rows' root mean
    square and multiplied by w_post (if given), by the gate ([cols] or [rows, cols], if given)
    and alpha, and added to the residual x: y.  h is y divided by its root mean square, times
    w_pre (None without w_pre): the next block's input.  stats [2, rows] float32 is for
    block_norm_backward.  out_y may be x, out_h may be o."""
    d = _block_norm((x, o, out_y, out_h), gate, w_post, w_pre, alpha, eps)
    y = torch.empty_like(x) if out_y is None else out_y
    h = None if w_pre is None else torch.empty_like(x) if out_h is None else out_h
    stats = torch.empty((2, x.shape[0]), device=x.device, dtype=torch.float32)
    check(lib().katsu_hip_block_norm_dev(ctypes.byref(d), _p(x), _p(o), _p(gate), _p(w_post),
                                         _p(w_pre), _p(y), _p(h), _p(stats), _stream()),
          "block_norm")
    return y, h, stats


def block_norm_backward(dy, dh, y, o, stats, gate=None, w_post=None, w_pre=None, alpha=1.0,
                        workspace=None):
    """(dx, do, dgate, dw_post, dw_pre) from dy, the gradient that reaches y otherwise, and dh,
    with block_norm's y and stats; None for operands that were not given (dh and y may then be
    None without w_pre)."""
    if w_pre is not None and (dh is None or y is None):
        raise ValueError("dh and y are needed with w_pre")
    d = _block_norm((dy, dh, y, o), gate, w_post, w_pre, alpha, 0.0)
    if (stats.dtype is not torch.float32 or stats.device != dy.device
            or stats.shape != (2, dy.shape[0]) or not stats.is_contiguous()):
        raise ValueError("stats must be what block_norm returned")
    dx, do = torch.empty_like(dy), torch.empty_like(dy)
    dgate, dw_post, dw_pre = (None if t is None else torch.empty_like(t)
                              for t in (gate, w_post, w_pre))
    check(lib().katsu_hip_block_norm_bwd_dev(
        ctypes.byref(d), _p(dy), _p(dh), _p(y), _p(o), _p(stats), _p(gate), _p(w_post), _p(w_pre),
        _p(dx), _p(do), _p(dgate), _p(dw_post), _p(dw_pre), *_workspace(workspace, dy.device),
        _stream()), "block_norm_backward")
    return dx, do, dgate, dw_post, dw_pre


def block_norm_workspace_bytes(dy):
    """Scratch that block_norm_backward needs for gradients of this shape."""
    d = _block_norm((dy,), None, None, None, 1.0, 0.0)
    nbytes = ctypes.c_size_t(0)
    check(lib().katsu_hip_block_norm_bwd_workspace(ctypes.byref(d), ctypes.byref(nbytes)),
          "block_norm_workspace")
    return nbytes.value


def clip_workspace_bytes(n):
    """Scratch that clip_grad_norm needs for n gradients."""
    nbytes = ctypes.c_size_t(0)
    check(lib().katsu_hip_clip_grad_norm_workspace(n, ctypes.byref(nbytes)), "clip_workspace")
    return nbytes.value


def clip_grad_norm(grads, max_norm, out=None, workspace=None):
    """The root of the sum of all squares of `grads` (a list of contiguous device tensors of
    either type), as a float32 device tensor [1]; each gradient times
    min(1, max_norm / (norm + 1e-6)) is written to `out` (in place if None).  No two of the tensors
    written may share memory.  `workspace`: an optional device tensor of clip_workspace_bytes();
    without it the library's own buffer is used."""
    n = len(grads)
    if n == 0:
        raise ValueError("no gradients")
    # Lists of one attribute each and array's buffers: the host side of 26 tensors takes 28 us so,
    # 44 with a check tensor by tensor and ctypes arrays.
    types, devs = [g.dtype for g in grads], {g.get_device() for g in grads}
    sizes, whole = [g.numel() for g in grads], [g.is_contiguous() for g in grads]
    ptrs = outs = array("Q", [g.data_ptr() for g in grads])
    same = True
    if out is not None and out is not grads:
        devs |= {o.get_device() for o in out}
        whole += [o.is_contiguous() for o in out]
        same = types == [o.dtype for o in out] and sizes == [o.numel() for o in out]
        outs = array("Q", [o.data_ptr() for o in out])
    if (not same or False in whole or len(devs) != 1 or -1 in devs
            or any(t not in _DTYPE for t in types)):
        raise ValueError("gradients and outputs must be contiguous float32 or bfloat16 tensors on "
                         "one device, each output of its gradient's size and type")
    norm = torch.empty(1, device=grads[0].device, dtype=torch.float32)
    kinds, counts = array("i", [_DTYPE[t] for t in types]), array("Q", sizes)
    check(lib().katsu_hip_clip_grad_norm_ws_dev(
        kinds.buffer_info()[0], ptrs.buffer_info()[0], outs.buffer_info()[0],
        counts.buffer_info()[0], n, max_norm, norm.data_ptr(),
        *_workspace(workspace, norm.device), _stream()), "clip_grad_norm")
    return norm


# ---- the ends of a language model, and the heads before its attention ----

def _at(t):
    return 0 if t is None else t.data_ptr()


def _operands(first, *ts):
    """float32 or bfloat16, all of the first one's type, on the current device: the launches go to its
    current stream.  (Type and device number are compared: a device object takes 0.1 us to make.)"""
    dt, dev = first.dtype, first.get_device()
    if dt not in _DTYPE or dev < 0:
        raise ValueError("float32 or bfloat16 device tensors expected")
    if dev != torch._C._cuda_getDevice():
        raise ValueError("operands must be on the current device")
    for t in ts:
        if t is not None and (t.dtype is not dt or t.get_device() != dev):
            raise ValueError("all operands must have one type and device")
    return _DTYPE[dt]


def _scratch(workspace, first, size_fn, d):
    """The caller's workspace, or one of torch's for this call: unlike the library's own buffer it
    belongs to the stream, or to the graph that is captured."""
    if workspace is None:
        nbytes = ctypes.c_size_t(0)
        check(size_fn(d, nbytes), "workspace")
        if nbytes.value == 0:
            return None, 0, 0
        workspace = first.new_empty(nbytes.value, dtype=torch.uint8)
        return workspace, workspace.data_ptr(), nbytes.value
    return (workspace, *_workspace(workspace, first.device))


def _rows(t, what):
    """A [rows, cols] tensor's row stride; its columns must be adjacent."""
    if t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1):
        raise ValueError(f"{what} must be [rows, cols] with adjacent columns")
    return t.stride(0)


def _embedding(table, out, ids, scale, beta):
    kind = _operands(table, out)
    strides = _rows(table, "the table"), _rows(out, "out")
    if out.shape[1] != table.shape[1] or table.shape[1] == 0:
        raise ValueError("out must have the table's columns, one at least")
    if beta not in (0.0, 1.0):
        raise ValueError("beta must be 0 or 1")
    _int32(ids, out.shape[0], table.device, "ids")
    return Embedding(kind, int(beta), out.shape[0], *table.shape, *strides, scale)


def embedding(ids, table, scale=1.0, out=None):
    """[T, C]: scale times the rows of table [V, C] that ids (int32 [T]) name; zeros where an id is
    not in [0, V), as for padding.  Rows of table and out may have any stride; they share no
    memory."""
    if out is None:
        out = table.new_empty((ids.numel(), table.shape[-1]))
    d = _embedding(table, out, ids, scale, 0.0)
    check(lib().katsu_hip_embedding_dev(d, _at(ids), _at(table), _at(out), _stream()),
          "embedding")
    return out


def embedding_backward(dout, ids, vocab, scale=1.0, out=None, beta=0.0, workspace=None):
    """The gradient of embedding's table [vocab, C] from dout [T, C]: each row the sum of its
    tokens' gradients, times scale; tokens with an id that is no row add nothing.  beta=1
    accumulates into `out` and leaves rows without a token as they are; out shares no memory with
    dout.  The same call gives the same bits.  `workspace`: an optional device tensor of
    embedding_workspace_bytes()."""
    if out is None:
        if beta != 0.0:
            raise ValueError("beta=1 needs the gradient that it accumulates into")
        out = dout.new_empty((vocab, dout.shape[-1]))
    if out.shape[0] != vocab:
        raise ValueError("out must have a row for each of the vocabulary")
    d = _embedding(out, dout, ids, scale, beta)
    keep, *ws = _scratch(workspace, dout, lib().katsu_hip_embedding_bwd_workspace, d)
    check(lib().katsu_hip_embedding_bwd_dev(d, _at(dout), _at(ids), _at(out), *ws,
                                            _stream()), "embedding_backward")
    return out


def embedding_workspace_bytes(tokens, vocab, cols, dtype):
    """Scratch that embedding_backward needs."""
    d = Embedding(_DTYPE[dtype], 0, tokens, vocab, cols, cols, cols, 1.0)
    nbytes = ctypes.c_size_t(0)
    check(lib().katsu_hip_embedding_bwd_workspace(ctypes.byref(d), ctypes.byref(nbytes)),
          "embedding_workspace")
    return nbytes.value


def _qk_norm_rotary(q, k, out_q, out_k, table, positions, w_q, w_k, eps, interleaved, *more):
    kind = _operands(q, k, out_q, out_k, w_q, w_k, *more)
    (q0, q1), (o0, o1) = _heads(q, "q"), _heads(out_q, "out_q")
    k0 = k1 = p0 = p1 = k_heads = length = rot = 0
    shape = q.shape
    tokens, heads, dim = shape
    if out_q.shape != shape or (k is None) != (out_k is None):
        raise ValueError("outputs must have the operands' shapes")
    if k is not None:
        (k0, k1), (p0, p1) = _heads(k, "k"), _heads(out_k, "out_k")
        k_tokens, k_heads, k_dim = shape = k.shape
        if out_k.shape != shape or k_tokens != tokens or k_dim != dim:
            raise ValueError("q and k must have the same tokens and channels, outputs their shapes")
    elif w_k is not None:
        raise ValueError("w_k goes with k")
    for w in (w_q, w_k):
        if w is not None and (w.shape != (dim,) or not w.is_contiguous()):
            raise ValueError("weights must be contiguous [channels]")
    if table is not None:
        if (table.dim() != 2 or table.dtype is not torch.float32 or not table.is_contiguous()
                or table.get_device() != q.get_device() or table.shape[1] == 0):
            raise ValueError("table must be contiguous float32 [length, channels that turn]")
        length, rot = table.shape
    elif positions is not None:
        raise ValueError("positions go with a table")
    if positions is not None:
        _int32(positions, tokens, q.device, "positions")
    return QkNormRotary(kind, bool(interleaved), tokens, heads, k_heads, dim, rot, length, q0, q1,
                        k0, k1, o0, o1, p0, p1, eps)


def qk_norm_rotary(q, k, table=None, positions=None, w_q=None, w_k=None, eps=1e-6,
                   interleaved=False, out_q=None, out_k=None):
    """(q', k'): each head of q and k [tokens, heads, channels] (k may be None) divided by its
    channels' root mean square, times w_q or w_k ([channels], None: no weight), then turned as
    rotary does by rows of `table` (None: not turned), in one pass and rounded once.  At most 512
    channels, adjacent; any token and head strides.  out_q may be q, and out_k k; otherwise they
    share no memory with an operand or each other."""
    out_q = torch.empty_like(q) if out_q is None else out_q
    if k is not None and out_k is None:
        out_k = torch.empty_like(k)
    d = _qk_norm_rotary(q, k, out_q, out_k, table, positions, w_q, w_k, eps, interleaved)
    check(lib().katsu_hip_qk_norm_rotary_dev(d, _at(q), _at(k), _at(w_q), _at(w_k), _at(table),
                                             _at(positions), _at(out_q), _at(out_k), _stream()),
          "qk_norm_rotary")
    return out_q, out_k


def qk_norm_rotary_backward(dq, dk, q, k, table=None, positions=None, w_q=None, w_k=None,
                            eps=1e-6, interleaved=False, out_q=None, out_k=None, workspace=None):
    """(dx_q, dx_k, dw_q, dw_k) from dq and dk, the gradients of qk_norm_rotary's outputs, and its
    operands; None for those that were not given.  out_q and out_k receive dx_q and dx_k; out_q may
    be dq or q, out_k dk or k; otherwise they share no memory with an operand or each other.
    `workspace`: an optional device tensor of qk_norm_rotary_workspace_bytes()."""
    out_q = torch.empty_like(q) if out_q is None else out_q
    if k is not None and out_k is None:
        out_k = torch.empty_like(k)
    d = _qk_norm_rotary(q, k, out_q, out_k, table, positions, w_q, w_k, eps, interleaved, dq, dk)
    if dq.shape != q.shape or (dk is None) != (k is None) or (k is not None
                                                              and dk.shape != k.shape):
        raise ValueError("gradients must have their operands' shapes")
    g = QkNormRotaryGrads(*_heads(dq, "dq"), *((0, 0) if dk is None else _heads(dk, "dk")))
    dw_q, dw_k = (None if w is None else torch.empty_like(w) for w in (w_q, w_k))
    keep, *ws = _scratch(workspace, q, lib().katsu_hip_qk_norm_rotary_bwd_workspace, d)
    check(lib().katsu_hip_qk_norm_rotary_bwd_dev(
        d, g, _at(dq), _at(dk), _at(q), _at(k), _at(w_q), _at(w_k), _at(table), _at(positions),
        _at(out_q), _at(out_k), _at(dw_q), _at(dw_k), *ws, _stream()), "qk_norm_rotary_backward")
    return out_q, out_k, dw_q, dw_k


def qk_norm_rotary_workspace_bytes(q, k):
    """Scratch that qk_norm_rotary_backward needs for operands of these shapes (k may be None)."""
    d = _qk_norm_rotary(q, k, q, k, None, None, None, None, 0.0, False)
    nbytes = ctypes.c_size_t(0)
    check(lib().katsu_hip_qk_norm_rotary_bwd_workspace(ctypes.byref(d), ctypes.byref(nbytes)),
          "qk_norm_rotary_workspace")
    return nbytes.value


def _distillation(logits, ids, teacher, temperature, out=None, dloss=None):
    kind = _operands(logits, out)
    strides = _rows(logits, "logits"), 0 if out is None else _rows(out, "out")
    rows, vocab = logits.shape
    if out is not None and out.shape != logits.shape:
        raise ValueError("out must have the logits' shape")
    if (ids.dim() != 2 or ids.shape[0] != rows or teacher.shape != ids.shape
            or ids.dtype is not torch.int32 or teacher.dtype not in _DTYPE
            or not ids.is_contiguous() or not teacher.is_contiguous()
            or not ids.get_device() == teacher.get_device() == logits.get_device()):
        raise ValueError("ids (int32) and teacher (float32 or bfloat16) must be contiguous "
                         "[rows, top] on the logits' device")
    if dloss is not None and (dloss.dtype is not torch.float32 or dloss.device != logits.device
                              or dloss.shape != (rows,)):
        raise ValueError("dloss must be float32 [rows] on the logits' device")
    return Distillation(kind, _DTYPE[teacher.dtype], rows, vocab, ids.shape[1],
                        *strides, 0 if dloss is None else dloss.stride(0), temperature)


def distillation(logits, ids, teacher, temperature=1.0):
    """(loss, stats): for each row of logits [rows, V] temperature^2 times the divergence of
    softmax(logits / temperature) from the teacher's softmax(teacher / temperature) over its top
    logits, teacher [rows, K] at the columns ids (int32 [rows, K], K at most 1024); entries with an
    id that is no column do not count.  loss [rows], float32.  K = 1 and temperature 1: the cross
    entropy with labels.  A row without an entry has loss 0.  stats [2, rows] float32 is for
    distillation_backward."""
    d = _distillation(logits, ids, teacher, temperature)
    loss = logits.new_empty(d.rows, dtype=torch.float32)
    stats = logits.new_empty((2, d.rows), dtype=torch.float32)
    check(lib().katsu_hip_distillation_dev(d, _at(logits), _at(ids), _at(teacher), _at(loss),
                                           _at(stats), _stream()), "distillation")
    return loss, stats


def distillation_backward(dloss, logits, ids, teacher, stats, temperature=1.0, out=None):
    """The gradient of the logits from dloss (float32 [rows], any stride) and distillation's operands
    and stats; zeros in rows without an entry.  `out` may be the logits; otherwise it shares no memory
    with them."""
    out = torch.empty_like(logits) if out is None else out
    d = _distillation(logits, ids, teacher, temperature, out, dloss)
    if (stats.dtype is not torch.float32 or stats.device != logits.device
            or stats.shape != (2, d.rows) or not stats.is_contiguous()):
        raise ValueError("stats must be what distillation returned")
    check(lib().katsu_hip_distillation_bwd_dev(d, _at(dloss), _at(logits), _at(ids), _at(teacher),
                                               _at(stats), _at(out), _stream()),
          "distillation_backward")
    return out


def distillation_step(logits, ids, teacher, dloss, temperature=1.0, out=None):
    """(loss, gradient of the logits) in one pass over them, where dloss (float32 [rows], any
    stride: what the sum or the mean of the losses gives each) is known beforehand.  `out`, the
    gradient, may be the logits; otherwise it shares no memory with them."""
    out = torch.empty_like(logits) if out is None else out
    d = _distillation(logits, ids, teacher, temperature, out, dloss)
    loss = logits.new_empty(d.rows, dtype=torch.float32)
    check(lib().katsu_hip_distillation_step_dev(d, _at(logits), _at(ids), _at(teacher), _at(dloss),
                                                _at(loss), _at(out), _stream()),
          "distillation_step")
    return loss, out
