"""Host entry points with the call signatures of the reference's generated host functions.

``softmax(x)``                       triton_generated/softmax/softmax.py:97-160
``lego_layer_norm(x, shape, w, b, eps)``  triton_generated/layernorm/layernorm.py:279-307, 407
``matmul(a, b, activation="")``      triton_generated/matmul/matmul_NTA_NTB.py:129-145
``lego_group_gemm_fn(group_A, group_B)``  triton_generated/grouped_gemm/grouped_gemm.py:120-162
``transpose(x)``                     the generated transpose programs have no callable
                                     (mlir_generated/transpose/transpose_smem_4096.mlir:2)

and, beside them, what stands between the projections of a transformer block: ``rotary``, ``attention`` and
``tree_attention``, which the reference has no counterpart of.

As in the reference, inputs are borrowed, outputs are allocated here with ``torch.empty``
and the kernel is enqueued on the current stream without synchronisation.  Tensors are
only carriers of device pointers: every call goes through the C ABI of liblego_hip.so.
"""
from __future__ import annotations

import contextlib
import ctypes
import math
import warnings

import torch

from . import runtime


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream():
    """The current stream's handle (an integer, or None for the null stream: what a ``c_void_p`` parameter takes);
    asked for on every call, since the caller may switch streams."""
    if _raw_stream is not None:      # without building a torch.cuda.Stream object
        return _raw_stream(torch.cuda.current_device()) or None
    return torch.cuda.current_stream().cuda_stream or None


def _ptr(t):
    """The tensor's address as an integer (None for an empty tensor's null pointer): a ``c_void_p`` parameter."""
    return t.data_ptr() or None


def _check(t, dtype, name, ndim=2):
    if not t.is_cuda:
        raise ValueError(f"{name} must live on the GPU")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if t.dim() != ndim:
        raise ValueError(f"{name} must have {ndim} dimensions")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


class _InPython:
    """In place of the module in C++: every call is Python's."""

    transpose = softmax = stencil = matmul = group = attention = tree = rotary = staticmethod(lambda *args: None)


_calls = None
_call = runtime.call


def _host():
    """The operators' host side in C++ (csrc/host_calls.cpp); each gives None for what it leaves to Python: other than plain GPU tensors,
    calls under a tracer, a mode or a transform, and calls that are refused.  A program that puts a function of its own in the place of
    ``runtime.call``, to record or time what is called, sees these operators' calls in it: they are all made in Python then."""
    global _calls
    if torch.compiler.is_compiling() or runtime.call is not _call:
        return _InPython
    if _calls is None:
        try:
            _calls = runtime.host_calls()
        except (FileNotFoundError, ImportError) as e:
            warnings.warn(f"the operators' host side runs in Python, some 3 us more a call: {e}", RuntimeWarning, stacklevel=3)
            _calls = _InPython
    return _calls


def transpose(x: torch.Tensor) -> torch.Tensor:
    """``x.T`` materialised: the ``rows x cols`` row-major input copied into the
    column-major layout of the same logical matrix."""
    out = _host().transpose(x)
    if out is not None:
        return out
    if x.element_size() not in (2, 4):
        raise ValueError("transpose moves 2-byte and 4-byte elements (float16, bfloat16, float32, int32, ...)")
    _check(x, x.dtype, "x")
    rows, cols = x.shape
    out = torch.empty((cols, rows), device=x.device, dtype=x.dtype)
    # the kernels move bits: the entry point is chosen by element size
    entry = "lego_hip_transpose_f32" if x.element_size() == 4 else "lego_hip_transpose_f16"
    runtime.call(entry, _ptr(x), _ptr(out), rows, cols, _stream())
    return out


_ROW_TAG = {torch.float16: "f16", torch.bfloat16: "bf16", torch.float32: "f32"}


def softmax(x: torch.Tensor, waves_per_row: int | None = None) -> torch.Tensor:
    """Row softmax of a 2-D fp16, bf16 or fp32 tensor."""
    if waves_per_row is None:
        y = _host().softmax(x)
        if y is not None:
            return y
    if x.dtype not in _ROW_TAG:
        raise ValueError("softmax supports float16, bfloat16 and float32")
    _check(x, x.dtype, "x")
    n_rows, n_cols = x.shape
    y = torch.empty_like(x)
    if waves_per_row is None:
        runtime.call(f"lego_hip_softmax_{_ROW_TAG[x.dtype]}", _ptr(x), _ptr(y), n_rows, n_cols, _stream())
    elif x.dtype != torch.float16:
        raise ValueError("waves_per_row is a tuning knob of the fp16 kernels")
    else:
        runtime.call("lego_hip_softmax_f16_wpr", _ptr(x), _ptr(y), n_rows, n_cols, waves_per_row, _stream())
    return y


def layer_norm_fwd(x, weight, bias, eps=1e-5, waves_per_row: int | None = None):
    """LayerNorm forward over the last dimension; returns ``(y, mean, rstd)``."""
    if x.dtype not in _ROW_TAG:
        raise ValueError("x must be float16, bfloat16 or float32")
    x_arg = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])      # every torch call here costs a microsecond
    _check(x_arg, x.dtype, "x")
    M, N = x_arg.shape
    _check(weight, x.dtype, "weight", ndim=1)
    _check(bias, x.dtype, "bias", ndim=1)
    if weight.shape[0] != N or bias.shape[0] != N:
        raise ValueError("weight and bias must have the size of the normalised dimension")
    if N * x.element_size() > 65536:
        # the reference's limit and message (layernorm.py:293-294)
        raise RuntimeError("This layer norm doesn't support feature dim >= 64KB.")
    y = torch.empty_like(x_arg)
    mean = torch.empty((M,), dtype=torch.float32, device=x.device)
    rstd = torch.empty((M,), dtype=torch.float32, device=x.device)
    args = (_ptr(x_arg), _ptr(y), _ptr(weight), _ptr(bias), _ptr(mean), _ptr(rstd), M, N, float(eps))
    if waves_per_row is None:
        runtime.call(f"lego_hip_layernorm_fwd_{_ROW_TAG[x.dtype]}", *args, _stream())
    elif x.dtype != torch.float16:
        raise ValueError("waves_per_row is a tuning knob of the fp16 kernels")
    else:
        runtime.call("lego_hip_layernorm_fwd_f16_wpr", *args, waves_per_row, _stream())
    return (y if x.dim() == 2 else y.view(x.shape)), mean, rstd


_bwd_workspace = {}      # (element tag, M, N) -> bytes of fp32 partial sums


def layer_norm_bwd(dy, x, weight, mean, rstd):
    """LayerNorm backward; returns ``(dx, dw, db)``.  fp16, bf16 or fp32 tensors, rows of up to 32768 elements."""
    if x.dtype not in _ROW_TAG:
        raise ValueError("x must be float16, bfloat16 or float32")
    tag = _ROW_TAG[x.dtype]
    x_arg = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    dy_arg = dy if dy.dim() == 2 and dy.is_contiguous() else dy.reshape(-1, dy.shape[-1]).contiguous()
    _check(x_arg, x.dtype, "x")
    _check(dy_arg, x.dtype, "dy")
    _check(weight, x.dtype, "weight", ndim=1)
    M, N = x_arg.shape
    if dy_arg.shape != x_arg.shape or weight.shape[0] != N:
        raise ValueError("dy must have the shape of x and weight the length of its rows")
    for name, stat in (("mean", mean), ("rstd", rstd)):
        _check(stat, torch.float32, name, ndim=1)       # the forward pass's fp32 statistics, one per row
        if stat.shape[0] != M or stat.device != x.device:
            raise ValueError(f"{name} must hold one float32 per row of x, on its device")
    need = _bwd_workspace.get((tag, M, N))
    if need is None:      # asked once per shape: the answer is a function of the shape alone
        size = ctypes.c_ulonglong(0)
        runtime.call("lego_hip_layernorm_bwd_workspace_bytes" if tag == "f16" else f"lego_hip_layernorm_bwd_{tag}_workspace_bytes",
                     M, N, ctypes.byref(size))
        if len(_bwd_workspace) >= 4096:
            _bwd_workspace.clear()
        need = _bwd_workspace[(tag, M, N)] = size.value
    # like the reference's wrapper, which allocates its partial buffers with torch (layernorm.py:381-383)
    workspace = torch.empty(need // 4, dtype=torch.float32, device=x.device)
    dx = torch.empty_like(x_arg)
    dw = torch.empty((N,), dtype=weight.dtype, device=x.device)
    db = torch.empty((N,), dtype=weight.dtype, device=x.device)
    runtime.call(f"lego_hip_layernorm_bwd_{tag}", _ptr(dy_arg), _ptr(x_arg), _ptr(weight), _ptr(mean), _ptr(rstd),
                 _ptr(dx), _ptr(dw), _ptr(db), _ptr(workspace), need, M, N, _stream())
    return (dx if x.dim() == 2 else dx.view(x.shape)), dw, db


class LEGOLayerNorm(torch.autograd.Function):
    """The node of ``lego_layer_norm`` in Python, for calls that the one in C++ leaves to it."""

    @staticmethod
    def forward(ctx, x, normalized_shape, weight, bias, eps):
        if tuple(normalized_shape) != (x.shape[-1],):
            raise ValueError("normalized_shape must be the last dimension of x")
        y, mean, rstd = layer_norm_fwd(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, bias, mean, rstd)
        ctx.eps = eps
        return y

    @staticmethod
    def backward(ctx, dy):
        x, w, b, m, v = ctx.saved_tensors
        dx, dw, db = layer_norm_bwd(dy, x, w, m, v)
        return dx, None, dw, db, None


_node_apply = None


def _load_node():
    """The node in C++, or, where it is not built or not for this torch, one that leaves every call to the node in Python (the same
    kernels, some 50 us more of host time a step), and says so."""
    global _node_apply
    try:
        _node_apply = runtime.layernorm_node().apply
    except (FileNotFoundError, ImportError) as e:
        warnings.warn(f"LayerNorm runs through its autograd node in Python: {e}", RuntimeWarning, stacklevel=3)
        _node_apply = lambda *args: None      # noqa: E731
    return _node_apply


def lego_layer_norm(x, normalized_shape, weight, bias, eps):
    """LayerNorm with the reference's signature and gradients (triton_generated/layernorm/layernorm.py:323-407).  Plain GPU
    tensors go through the node in C++ (csrc/layernorm_node.cpp); subclasses, dual tensors, calls under a tracer, a mode or a
    transform, and calls that are refused, through the one above."""
    if not torch.compiler.is_compiling():
        y = (_node_apply or _load_node())(x, normalized_shape, weight, bias, eps)
        if y is not None:
            return y
    return LEGOLayerNorm.apply(x, normalized_shape, weight, bias, eps)


_GEMM_ENTRY = {torch.float16: "lego_hip_gemm_f16_ex", torch.bfloat16: "lego_hip_gemm_bf16_ex"}
_FP8_FORMAT = {torch.float8_e4m3fn: 0, torch.float8_e5m2: 1}


def _operand(t, name):
    """``(storage tensor, transposed?)`` of a 2-D fp16/bf16 operand that is contiguous either as
    given or as its transpose (the reference's TA/TB variants pass ``x.T`` views)."""
    if not t.is_cuda or (t.dtype not in _GEMM_ENTRY and t.dtype not in _FP8_FORMAT) or t.dim() != 2:
        raise ValueError(f"{name} must be a 2-D float16, bfloat16 or float8 GPU tensor")
    if t.is_contiguous():
        return t, 0
    if t.t().is_contiguous():
        return t.t(), 1
    raise ValueError(f"{name} must be contiguous or the transpose of a contiguous tensor")


_gemm_workspace = {}      # (M, N, K, ta, tb, ...) -> bytes of workspace that the product uses


def _ask_workspace(entry, known, shape):
    """The size for a shape seen for the first time, kept in ``known``."""
    size = ctypes.c_ulonglong(0)
    runtime.call(entry, *shape, ctypes.byref(size))
    if len(known) >= 4096:
        known.clear()
    known[shape] = size.value
    return size.value


def matmul(a: torch.Tensor, b: torch.Tensor, activation: str = "", out_dtype=torch.float16) -> torch.Tensor:
    """``act(a @ b)`` for fp16, bf16 or 8-bit floating-point operands of any shape, each row-major or
    column-major (a ``.T`` view), fp32 accumulation, row-major fp16 result: the reference's ``matmul``
    allocates a float16 result whatever its operands' type (matmul_sympy.py:129-145, its fp8 path
    :346-364).  ``out_dtype=torch.bfloat16`` with bfloat16 operands keeps their type instead."""
    c = _host().matmul(a, b, activation, out_dtype)
    if c is not None:
        return c
    if activation not in ("", "leaky_relu"):
        raise NotImplementedError(f"activation {activation!r} is not generated by this build")
    a_store, ta = _operand(a, "a")
    b_store, tb = _operand(b, "b")
    M, K = a.shape
    K2, N = b.shape
    if K != K2:
        raise ValueError("Incompatible dimensions")
    if a.dtype != b.dtype:
        raise ValueError("a and b must have the same dtype")
    if a.dtype in _FP8_FORMAT:
        c = torch.empty((M, N), device=a.device, dtype=torch.float16)
        if N % 16 or (M if ta else K) % 16 or (tb and K % 16):
            entry = "lego_hip_gemm_fp8_padded"      # rows that are not whole 16-byte chunks: zero-padded copies where they gain
        else:
            entry = "lego_hip_gemm_fp8_ex_ws"
        need = _gemm_workspace.get((M, N, K, ta, tb, 1))
        if need is None:
            need = _ask_workspace("lego_hip_gemm_layout_workspace_bytes", _gemm_workspace, (M, N, K, ta, tb, 1))
        if need:
            workspace = torch.empty(need, dtype=torch.uint8, device=a.device)
            runtime.call(entry, _ptr(a_store), _ptr(b_store), _ptr(c), M, N, K, ta, tb,
                         1 if activation else 0, _FP8_FORMAT[a.dtype], _ptr(workspace), need, _stream())
            return c
        runtime.call("lego_hip_gemm_fp8_ex", _ptr(a_store), _ptr(b_store), _ptr(c), M, N, K, ta, tb,
                     1 if activation else 0, _FP8_FORMAT[a.dtype], _stream())
        return c
    if out_dtype not in (torch.float16, a.dtype):
        raise ValueError("out_dtype must be float16 or the operands' type")
    entry = "lego_hip_gemm_bf16_f16_ex" if (a.dtype, out_dtype) == (torch.bfloat16, torch.float16) else _GEMM_ENTRY[a.dtype]
    if ta and M % 8 and (M * K >= 65536 or (K >= 384 and not (N % 8 or K % 8)) or (tb and M <= 16 and N >= 1024 and 1400 <= K <= 1984)):
        # a column-major A whose columns (M elements) are not whole 16-byte chunks is outside the tiled kernels unless the product
        # runs on copies anyway: store it row-major first (one pass with the transpose kernels; by elements / row-major first:
        # 33 x 256 x 256 13 / 15 us, 7 x 512 x 512 22 / 16, 3 x 1024 x 8192 323 / 19).  Where copies take it as well: first for the kernel for
        # few rows where the chain of K is long and not yet split (2 x 2049 x 801 20 / 26, 1602 29 / 26, 1922 33 / 26, 2102 23 / 27)
        a_store, ta = transpose(a_store), 0
    c = torch.empty((M, N), device=a.device, dtype=out_dtype)
    # products of few tiles (a skinny operand, a long K) are split along K when there is room for the partial sums;
    # shapes whose operand rows are not whole 16-byte chunks run on zero-padded copies in the workspace
    need = _gemm_workspace.get((M, N, K, ta, tb, 2))
    if need is None:
        need = _ask_workspace("lego_hip_gemm_layout_workspace_bytes", _gemm_workspace, (M, N, K, ta, tb, 2))
    if need:
        workspace = torch.empty(need // 4, dtype=torch.float32, device=a.device)
        element = 0 if a.dtype == torch.float16 else 4 if out_dtype == torch.float16 else 1
        runtime.call("lego_hip_gemm_ex_ws", element, _ptr(a_store), _ptr(b_store), _ptr(c), M, N, K, ta, tb,
                     1 if activation else 0, _ptr(workspace), need, _stream())
        return c
    runtime.call(entry, _ptr(a_store), _ptr(b_store), _ptr(c), M, N, K, ta, tb, 1 if activation else 0, _stream())
    return c


_group_apart = {}      # sizes of a call's problems -> those that are products of their own


def _problems_apart(sizes):
    """Asked once for a list of sizes: the answer is a function of the sizes alone."""
    groups = len(sizes) // 3
    flags = (ctypes.c_int * groups)()
    sz, size, limit = (ctypes.c_int * len(sizes))(*sizes), ctypes.c_ulonglong(0), ctypes.c_int(0)
    runtime.call("lego_hip_grouped_gemm_f16_room", sz, groups, ctypes.byref(size), ctypes.byref(limit))
    if not limit.value:      # otherwise in parts, in the one launch
        runtime.call("lego_hip_grouped_gemm_f16_apart", sz, groups, flags)
    if len(_group_apart) >= 1024:
        _group_apart.clear()
    apart = _group_apart[sizes] = frozenset(g for g in range(groups) if flags[g])
    return apart


def lego_group_gemm_fn(group_A, group_B):
    """One launch for a list of independent GEMMs; returns the list of results."""
    group_C = _host().group(group_A, group_B)
    if group_C is not None:
        return group_C
    if len(group_A) != len(group_B):
        raise ValueError("group_A and group_B must have the same length")
    # Problems whose rows are not whole 16-byte chunks run on zero-padded copies in a workspace; those whose long chains the other
    # problems leave alone run on their own.
    sizes, ragged, deep = [], False, False
    for a, b in zip(group_A, group_B):
        _check(a, torch.float16, "A")
        _check(b, torch.float16, "B")
        M, K = a.shape
        depth, N = b.shape
        if K != depth:
            raise ValueError("Incompatible dimensions")
        sizes += [M, N, K]
        if N % 8 or K % 8:
            ragged = True
            deep = deep or K > 1984
    if ragged and len(group_A) == 1:      # 1000 x 1001 x 1002 24 us, in a grouped launch 29
        return [matmul(group_A[0], group_B[0])]
    if deep:
        key = tuple(sizes)
        apart = _group_apart.get(key)
        if apart is None:
            apart = _problems_apart(key)
        if apart:
            rest = [g for g in range(len(group_A)) if g not in apart]
            together = iter(_grouped([group_A[g] for g in rest], [group_B[g] for g in rest],
                                     [s for g in rest for s in sizes[3 * g:3 * g + 3]]) if rest else ())
            return [matmul(group_A[g], group_B[g]) if g in apart else next(together) for g in range(len(group_A))]
    return _grouped(group_A, group_B, sizes)


def _grouped(group_A, group_B, sizes):
    """Checked problems, all in the grouped launch."""
    groups = len(group_A)
    group_C = [torch.empty((sizes[3 * g], sizes[3 * g + 1]), device=a.device, dtype=a.dtype) for g, a in enumerate(group_A)]
    arr = ctypes.c_void_p * groups
    pa = arr(*[t.data_ptr() for t in group_A])
    pb = arr(*[t.data_ptr() for t in group_B])
    pc = arr(*[t.data_ptr() for t in group_C])
    sz = (ctypes.c_int * (3 * groups))(*sizes)
    size, limit = ctypes.c_ulonglong(0), ctypes.c_int(0)
    runtime.call("lego_hip_grouped_gemm_f16_room", sz, groups, ctypes.byref(size), ctypes.byref(limit))
    if size.value:
        workspace = torch.empty(size.value // 2, dtype=torch.float16, device=group_C[0].device)
        runtime.call("lego_hip_grouped_gemm_f16_ws", pa, pb, pc, sz, groups, _ptr(workspace), size.value, _stream())
        return group_C
    runtime.call("lego_hip_grouped_gemm_f16", pa, pb, pc, sz, groups, _stream())
    return group_C


def needleman_wunsch(reference: torch.Tensor, matrix: torch.Tensor, penalty: int) -> torch.Tensor:
    """Fills the ``(n+1) x (n+1)`` int32 score ``matrix`` in place (its first row and column are the
    borders) from the substitution scores ``reference``; returns ``matrix``.  The reference's
    benchmark is a whole program (benchmarks/cuda/nw/needle.cu:165-260) with no host callable."""
    _check(reference, torch.int32, "reference")
    _check(matrix, torch.int32, "matrix")
    if reference.shape != matrix.shape or matrix.shape[0] != matrix.shape[1]:
        raise ValueError("reference and matrix must be square and of the same shape")
    n = matrix.shape[0] - 1
    size = ctypes.c_ulonglong(0)
    runtime.call("lego_hip_nw_i32_workspace_bytes", n, ctypes.byref(size))
    workspace = torch.empty(size.value // 8, dtype=torch.int64, device=matrix.device) if size.value else None
    runtime.call("lego_hip_nw_i32_ws", _ptr(reference), _ptr(matrix), n, int(penalty),
                 None if workspace is None else _ptr(workspace), size.value, _stream())
    return matrix


def _stencil(entry, x, c, radius, bricks, out):
    if out is None:
        got = _host().stencil(x, c, radius, bricks, c.dim() == 3)
        if got is not None:
            return got
    _check(x, torch.float32, "x", ndim=3)
    _check(c, torch.float32, "c", ndim=c.dim())
    n = x.shape[0]
    if x.shape != (n, n, n):
        raise ValueError("x must be a cube")
    if out is None:      # the kernel writes the boundary's zeros as well: no pass of its own for them
        out, entry = torch.empty_like(x), entry + "_zeros"
    else:
        _check(out, torch.float32, "out", ndim=3)
        if out.shape != x.shape or out.device != x.device:
            raise ValueError("out must have the shape and device of x")
        if out.data_ptr() == x.data_ptr():
            raise ValueError("out must not alias x")
    runtime.call(entry, _ptr(x), _ptr(out), _ptr(c), n, int(radius), 1 if bricks else 0, _stream())
    return out


def stencil_f3d(x, c, radius=1, bricks=False, out=None):
    """Dense ``(2*radius+1)^3`` stencil with the ``8 x 8 x 8`` coefficient cube ``c``; ``x`` holds the
    ``n^3`` points row-major, or brick by brick when ``bricks`` is set (``x.view(-1)`` is the
    storage either way).  Boundary points keep the value of ``out`` (zeros by default, as the
    reference program's ``cudaMemset``, benchmarks/cuda/bricks/main_tmp.cu:160-163)."""
    if c.shape != (8, 8, 8):
        raise ValueError("c must be 8 x 8 x 8")
    return _stencil("lego_hip_stencil_f3d_f32", x, c, radius, bricks, out)


def stencil_laplacian(x, c, radius=1, bricks=False, out=None):
    """Star stencil ``c[0]*x + sum_a c[a]*(six neighbours at distance a)``; ``c`` has at least
    ``radius + 1`` entries."""
    if c.dim() != 1 or c.shape[0] < radius + 1:
        raise ValueError("c must hold radius + 1 coefficients")
    return _stencil("lego_hip_stencil_laplacian_f32", x, c, radius, bricks, out)


def lud(m: torch.Tensor) -> torch.Tensor:
    """LU decomposition without pivoting, in place; returns ``m`` holding L below the diagonal
    (unit diagonal implied) and U on and above it (benchmarks/cuda/lud/lud.cu: a whole program,
    no host callable)."""
    _check(m, torch.float32, "m")
    if m.shape[0] != m.shape[1]:
        raise ValueError("m must be square")
    runtime.call("lego_hip_lud_f32", _ptr(m), m.shape[0], _stream())
    return m


# Attention.  Tensors are [batch, token, head, element]; a query head reads key head h // (query heads / key heads).

_ATTENTION_ELEMENT = {torch.float16: 0, torch.bfloat16: 1}
MAX_HEAD = 128      # head elements that the attention kernels take, in whole eights
_MOST_PITCH = (1 << 24) - 256      # elements between tokens: a tile of 64 within 2 GiB


def _on(t):
    """The device of ``t`` as the current one: streams and launches are the current device's."""
    if t.device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(t.device)


def _strides(t):
    """Elements between batches, tokens and heads; 0 where there is one of them."""
    return [st if n > 1 else 0 for st, n in zip(t.stride(), t.shape[:3])]


def _in_chunks(t):
    """``t`` as the attention kernels read it: whole 16-byte chunks.  Slices of a fused projection are; other layouts are copied."""
    if (t.shape[3] == 1 or t.stride(3) == 1) and t.data_ptr() % 16 == 0:
        st = _strides(t)
        if not (st[0] % 8 or st[1] % 8 or st[2] % 8) and st[1] <= _MOST_PITCH:
            return t
    return t.clone(memory_format=torch.contiguous_format)


def _cache_in_chunks(t):
    """A cache is never copied: it is what the program lays out once."""
    st = _strides(t)
    if t.stride(3) != 1 or t.data_ptr() % 16 or st[0] % 8 or st[1] % 8 or st[2] % 8:
        raise ValueError("the caches must have elements one apart, and bases and strides in whole 16 bytes")
    return t


def _check_qkv(q, k, v, cache=False):
    for name, t in (("q", q), ("k", k), ("v", v)):
        if not t.is_cuda:
            raise ValueError(f"{name} must live on the GPU")
        if t.dtype not in _ATTENTION_ELEMENT:
            raise ValueError(f"{name} must be float16 or bfloat16, got {t.dtype}")
        if t.dim() != 4:
            raise ValueError(f"{name} must be [batch, token, head, element]")
        if t.dtype != q.dtype or t.device != q.device:
            raise ValueError("q, k and v must have the same dtype and device")
    if k.shape != v.shape:
        raise ValueError("k and v must have the same shape")
    if (k.shape[0] != q.shape[0] and not cache) or k.shape[3] != q.shape[3]:
        raise ValueError("q and k must have the same batch and head size")
    if k.shape[2] == 0 or q.shape[2] % k.shape[2]:
        raise ValueError("the query heads must be a multiple of the key heads")
    if q.shape[3] % 8 or not 8 <= q.shape[3] <= MAX_HEAD:
        raise ValueError(f"heads of 8, 16, ... {MAX_HEAD} elements, got {q.shape[3]}")


def _vector(t, name, dtype, shape, device):
    """A small tensor beside the operands, contiguous, or None."""
    if t is None:
        return None
    if t.dtype != dtype or t.device != device or tuple(t.shape) != shape:
        raise ValueError(f"{name} must be {dtype} of shape {list(shape)} on {device}")
    if t.requires_grad:
        raise ValueError(f"{name} has no gradient here")
    return t.contiguous()


def _check_mask(q, k, causal, scale, softcap, slopes, documents, prefix):
    """``(slopes, documents, prefix, scale, softcap)`` as the entry points take them."""
    scale = 1.0 / math.sqrt(q.shape[3]) if scale is None else float(scale)
    softcap = float(softcap or 0.0)
    if not math.isfinite(scale):
        raise ValueError("scale must be finite")
    if not (0.0 <= softcap < math.inf):
        raise ValueError("softcap must be positive, or 0 for none")
    if prefix is not None and not causal:
        raise ValueError("a prefix goes with a causal mask")
    if documents is not None and q.shape[1] > k.shape[1]:
        raise ValueError("documents are the keys', which the queries are the last of")
    return (_vector(slopes, "slopes", torch.float32, (q.shape[2],), q.device),
            _vector(documents, "documents", torch.int32, (k.shape[0], k.shape[1]), q.device),
            _vector(prefix, "prefix", torch.int32, (q.shape[0],), q.device), scale, softcap)


def _longs(values):
    return (ctypes.c_longlong * len(values))(*values)


def _optional(t):
    return None if t is None else t.data_ptr()


def _attention_room(sizes, documents, backward, device):
    size = ctypes.c_ulonglong(0)
    runtime.call("lego_hip_attention_workspace_bytes", sizes, documents, backward, ctypes.byref(size))
    return (torch.empty(size.value, dtype=torch.uint8, device=device) if size.value else None), size.value


def attention_fwd(q, k, v, causal=False, scale=None, softcap=0.0, slopes=None, documents=None, prefix=None, with_rest=False):
    """Attention without its gradient; returns ``(out, lse)``, with the fp32 logarithm of every query's sum of exponentials,
    ``[batch, head, query]`` (-inf for a query that sees no key), and ``with_rest`` what rounding took from ``out`` too, in a tensor like it.  Arguments as
    ``attention`` has them."""
    _check_qkv(q, k, v)
    slopes, documents, prefix, scale, softcap = _check_mask(q, k, causal, scale, softcap, slopes, documents, prefix)
    batch, queries, heads, head = q.shape
    out = torch.empty((batch, queries, heads, head), dtype=q.dtype, device=q.device)
    lse = torch.empty((batch, heads, queries), dtype=torch.float32, device=q.device)
    rest = torch.empty_like(out) if with_rest else None
    back = (out, lse, rest) if with_rest else (out, lse)
    if out.numel() == 0:
        return back
    if k.shape[1] == 0:
        out.zero_(), lse.fill_(-math.inf)
        if with_rest:
            rest.zero_()
        return back
    with _on(q):
        q, k, v = _in_chunks(q), _in_chunks(k), _in_chunks(v)
        sizes = _longs((batch, queries, k.shape[1], heads, k.shape[2], head))
        workspace, room = _attention_room(sizes, 1, 0, q.device) if documents is not None else (None, 0)
        runtime.call("lego_hip_attention_fwd", _ptr(q), _ptr(k), _ptr(v), _ptr(out), _optional(rest), _ptr(lse), sizes,
                     _longs(_strides(q) + _strides(k) + _strides(v) + _strides(out)), scale, softcap, _optional(slopes), _optional(documents),
                     _optional(prefix), 1 if causal else 0, _ATTENTION_ELEMENT[q.dtype], _optional(workspace), room, _stream())
    return back


def attention_bwd(dout, q, k, v, out, lse, causal=False, scale=None, softcap=0.0, slopes=None, documents=None, prefix=None, rest=None):
    """The gradients ``(dq, dk, dv)`` from that of ``out``, with ``out`` and ``lse`` of ``attention_fwd`` and its arguments; with ``rest`` the rounding of
    ``out`` is no part of their error.  Sums are in fp32 and in a fixed order: the same inputs give the same bits."""
    _check_qkv(q, k, v)
    slopes, documents, prefix, scale, softcap = _check_mask(q, k, causal, scale, softcap, slopes, documents, prefix)
    batch, queries, heads, head = q.shape
    for name, t in (("dout", dout), ("out", out), ("rest", out if rest is None else rest)):
        if t.shape != q.shape or t.dtype != q.dtype or t.device != q.device:
            raise ValueError(f"{name} must have the shape, dtype and device of q")
    if tuple(lse.shape) != (batch, heads, queries) or lse.dtype != torch.float32 or lse.device != q.device or not lse.is_contiguous():
        raise ValueError("lse must be attention_fwd's")
    dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
    if q.numel() == 0 or k.numel() == 0:
        return dq.zero_(), dk.zero_(), dv.zero_()
    with _on(q):
        dout, q, k, v = (_in_chunks(t) for t in (dout, q, k, v))
        out, rest = _in_chunks(out.contiguous()), None if rest is None else _in_chunks(rest.contiguous())
        sizes = _longs((batch, queries, k.shape[1], heads, k.shape[2], head))
        workspace, room = _attention_room(sizes, documents is not None, 1, q.device)
        strides = [st for t in (q, k, v, out, dout, dq, dk, dv) for st in _strides(t)]
        runtime.call("lego_hip_attention_bwd", _ptr(dout), _ptr(q), _ptr(k), _ptr(v), _ptr(out), _optional(rest), _ptr(lse), _ptr(dq), _ptr(dk), _ptr(dv), sizes,
                     _longs(strides), scale, softcap, _optional(slopes), _optional(documents), _optional(prefix), 1 if causal else 0,
                     _ATTENTION_ELEMENT[q.dtype], _optional(workspace), room, _stream())
    return dq, dk, dv


class _Once(torch.autograd.Function):
    """Gradients whose own gradient may be asked for: it is an error and not zero by what they came from."""

    @staticmethod
    def forward(ctx, name, count, *tensors):
        ctx.name = name
        return tuple(t.view_as(t) for t in tensors[:count])

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(f"{ctx.name} has no second derivative")


def _once(name, grads, *sources):
    return _Once.apply(name, len(grads), *grads, *sources) if torch.is_grad_enabled() else grads


class LEGOAttention(torch.autograd.Function):
    """The node of ``attention``."""

    @staticmethod
    def forward(ctx, q, k, v, causal, scale, softcap, slopes, documents, prefix):
        out, lse, rest = attention_fwd(q, k, v, causal, scale, softcap, slopes, documents, prefix, with_rest=True)
        ctx.save_for_backward(q, k, v, out, lse, slopes, documents, prefix, rest)
        ctx.how = (causal, scale, softcap)
        return out

    @staticmethod
    def backward(ctx, dout):
        q, k, v, out, lse, slopes, documents, prefix, rest = ctx.saved_tensors
        with torch.no_grad():
            grads = attention_bwd(dout, q, k, v, out, lse, *ctx.how, slopes, documents, prefix, rest)
        return _once("attention", grads, q, k, v, dout) + (None,) * 6


def attention(q, k, v, causal=False, scale=None, softcap=0.0, slopes=None, documents=None, prefix=None):
    """``softmax(s) v`` with gradients of q, k and v; fp16 or bf16, fp32 softmax and sums.

    q is ``[batch, queries, heads, element]``, k and v ``[batch, keys, key heads, element]`` (the heads a multiple of the key heads, each
    shared by its group; a head of 8, 16, ... 128 elements); slices of a fused projection are read where they lie.
    ``s = scale * q.k`` (default ``1/sqrt(element)``), then ``softcap * tanh(s / softcap)``, then less ``slopes[head] * |distance|`` (fp32, no gradient).
    Query i stands at position ``i + keys - queries``.  It sees the keys that are no later where ``causal``, and the first
    ``prefix[batch]`` (int32) whatever their place; of those the ones of its own document, ``documents`` (int32 ``[batch, keys]``; a negative
    number is padding, which sees and is seen by nothing, whatever it holds).  A query that sees nothing gives zeros, and takes and gives no gradient.
    A NaN or infinity in a key or value reaches the queries that see it, and may reach others within 64 positions of those.

    There is no second derivative: asking for one raises.  Inside a captured graph call ``attention_fwd`` and ``attention_bwd``: autograd's own bookkeeping of leaves is not made for it."""
    out = _host().attention(q, k, v, causal, scale, softcap, slopes, documents, prefix)
    if out is not None:
        return out
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return LEGOAttention.apply(q, k, v, causal, scale, softcap, slopes, documents, prefix)
    return attention_fwd(q, k, v, causal, scale, softcap, slopes, documents, prefix)[0]


def tree_attention(q, k, v, k_cache, v_cache, pages, lengths, tree=None, scale=None, softcap=0.0, slopes=None, positions=None):
    """Attention of drafted tokens over a paged cache, without gradients: one drafted token a sequence is a step of ordinary decoding, more are a chain
    or a tree to be verified.  fp16 or bf16, fp32 softmax and sums; any lengths side by side.

    q is ``[batch, draft, heads, element]``, k and v, the drafts' own, ``[batch, draft, key heads, element]``; the caches are
    ``[page, row, key heads, element]``, pages of any number of rows.  Key i of sequence b lies in row ``i % rows`` of page ``pages[b, i // rows]`` (int32
    ``[batch, width]``; a number that is no page's stands for keys that are not there), for i below ``lengths[b]`` (int32 ``[batch]``, at most ``width * rows``).
    A draft sees all cached keys of its sequence and the drafts that ``tree`` (bool ``[draft, draft]`` or ``[batch, draft, draft]``: which one, a row, sees which) shows it; without
    ``tree`` itself and the earlier ones.  With k and v None it sees the cache alone.  Scores are ``attention``'s; the distances of ``slopes`` go by ``positions`` (int32
    ``[batch, draft]``, a cached key's being its number; default ``lengths[b] + draft``).  A draft that sees nothing gives zeros."""
    out = _host().tree(q, k, v, k_cache, v_cache, pages, lengths, tree, scale, softcap, slopes, positions)
    if out is not None:
        return out
    if (k is None) != (v is None):
        raise ValueError("k and v go together")
    _check_qkv(q, *((k_cache, v_cache) if k is None else (k, v)), cache=k is None)
    if k is not None:
        if k.shape[1] != q.shape[1]:
            raise ValueError("q, k and v must have the same drafts")
        if k_cache.shape != v_cache.shape or k_cache.dim() != 4 or k_cache.shape[2:] != k.shape[2:] or any(t.dtype != q.dtype or t.device != q.device for t in (k_cache, v_cache)):
            raise ValueError("the caches must be [page, row, key head, element] of k's heads, dtype and device")
    batch, drafts, heads, head = q.shape
    count, page, key_heads = k_cache.shape[:3]
    scale = 1.0 / math.sqrt(head) if scale is None else float(scale)
    softcap = float(softcap or 0.0)
    if not math.isfinite(scale) or not 0.0 <= softcap < math.inf:
        raise ValueError("scale must be finite, and softcap positive, or 0 for none")
    if pages.dim() != 2:
        raise ValueError("pages must be [batch, width]")
    width = pages.shape[1]
    pages = _vector(pages, "pages", torch.int32, (batch, width), q.device)
    lengths = _vector(lengths, "lengths", torch.int32, (batch,), q.device)
    slopes = _vector(slopes, "slopes", torch.float32, (heads,), q.device)
    if positions is not None and slopes is None:
        raise ValueError("positions are what slopes go by")
    positions = _vector(positions, "positions", torch.int32, (batch, drafts), q.device)
    if tree is not None:
        if k is None:
            raise ValueError("a tree is of drafts: it takes k and v")
        tree = _vector(tree, "tree", torch.bool, (drafts, drafts) if tree.dim() == 2 else (batch, drafts, drafts), q.device)
        if slopes is not None and positions is None:
            raise ValueError("in a tree, slopes take the drafts' positions")
    out = torch.empty((batch, drafts, heads, head), dtype=q.dtype, device=q.device)
    if out.numel() == 0:
        return out
    if count * page * width == 0:      # no cache: the drafts among themselves
        if k is None:
            return out.zero_()
        k, v = _in_chunks(k), _in_chunks(v)
        k_cache, v_cache, pages, count, page, width = k, v, torch.full((batch, 1), -1, dtype=torch.int32, device=q.device), 1, 1, 1
    with _on(q):
        q, k_cache, v_cache = _in_chunks(q), _cache_in_chunks(k_cache), _cache_in_chunks(v_cache)
        if k is not None:
            k, v = _in_chunks(k), _in_chunks(v)
        sizes = _longs((batch, drafts, heads, key_heads, head, page, count, width))
        size = ctypes.c_ulonglong(0)
        runtime.call("lego_hip_tree_attention_workspace_bytes", sizes, ctypes.byref(size))
        workspace = torch.empty(size.value, dtype=torch.uint8, device=q.device) if size.value else None
        none = [0, 0, 0]
        strides = _longs(_strides(q) + (none if k is None else _strides(k)) + (none if v is None else _strides(v)) + _strides(k_cache) + _strides(v_cache) + _strides(out)
                         + [0 if tree is None or tree.dim() == 2 else drafts * drafts])
        runtime.call("lego_hip_tree_attention", _ptr(q), _optional(k), _optional(v), _ptr(k_cache), _ptr(v_cache), _ptr(out), _ptr(pages), _ptr(lengths), _optional(tree),
                     _optional(slopes), _optional(positions), sizes, strides, scale, softcap, _ATTENTION_ELEMENT[q.dtype], _optional(workspace), size.value, _stream())
    return out


_ROTARY_ELEMENT = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
MAX_ROTARY_PART = 256


def rotary_frequencies(part, base=10000.0, stretch=1.0, original=None, slow=1.0, fast=32.0, device="cuda"):
    """What ``rotary`` multiplies positions with: ``base ** (-2 i / part)`` radians a position for the ``part / 2`` pairs of a head, in float64.

    For contexts ``stretch`` times as long as the ``original`` positions that a model was trained on: frequencies that make fewer than ``slow`` turns over the
    original length are divided by ``stretch``, those of more than ``fast`` turns are kept, and between the two the division comes in
    linearly with the turns.  Without ``original`` all are divided."""
    if part < 2 or part % 2 or part > MAX_ROTARY_PART:
        raise ValueError(f"part must be even, from 2 to {MAX_ROTARY_PART}")
    if not (base > 0 and stretch > 0):
        raise ValueError("base and stretch must be positive")
    radians = float(base) ** (-torch.arange(0, part, 2, dtype=torch.float64) / part)
    if stretch != 1.0:
        keep = torch.zeros_like(radians)
        if original is not None:
            if not fast > slow:
                raise ValueError("fast must be above slow")
            keep = ((original * radians / (2 * math.pi) - slow) / (fast - slow)).clamp(0.0, 1.0)
        radians = radians * (keep + (1.0 - keep) / stretch)
    return radians.to(device)


def _rotary(q, k, positions, frequencies, interleaved, magnitude, inverse):
    """Checked tensors through the kernel; ``k`` may be None."""
    batch, tokens, heads, head = q.shape
    outs = [None if t is None else torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k)]
    key_heads = 0 if k is None else k.shape[2]
    if key_heads == 0 or outs[1].numel() == 0:
        if q.numel() == 0:
            return outs
        k, key_heads = None, 0
    elif q.numel() == 0:      # the keys alone, in the queries' place
        outs[1] = _rotary(k, None, positions, frequencies, interleaved, magnitude, inverse)[0]
        return outs
    with _on(q):
        ts = [t if t is None or head == 1 or t.stride(3) == 1 else t.contiguous() for t in (q, k)]
        strides = []
        for t in (ts[0], ts[1], outs[0], outs[1] if k is not None else None):
            strides += [0, 0, 0] if t is None else _strides(t)
        strides += [st if n > 1 else 0 for st, n in zip(positions.stride(), positions.shape)]
        runtime.call("lego_hip_rotary", _ptr(ts[0]), None if k is None else _ptr(ts[1]), _ptr(outs[0]), None if k is None else _ptr(outs[1]), _ptr(positions),
                     _ptr(frequencies), _longs((batch, tokens, heads, key_heads, head, 2 * frequencies.shape[0])), _longs(strides), 1 if interleaved else 0,
                     magnitude, inverse, _ROTARY_ELEMENT[q.dtype], 1 if positions.dtype == torch.int64 else 0, _stream())
    return outs


class LEGORotary(torch.autograd.Function):
    """The node of ``rotary``: its gradient is the turn back."""

    @staticmethod
    def forward(ctx, q, k, positions, frequencies, interleaved, magnitude):
        ctx.save_for_backward(positions, frequencies)
        ctx.how = (interleaved, magnitude)
        ctx.set_materialize_grads(False)
        return tuple(_rotary(q, k, positions, frequencies, interleaved, magnitude, 0))

    @staticmethod
    def backward(ctx, dq, dk):
        positions, frequencies = ctx.saved_tensors
        given = [t for t in (dq, dk) if t is not None]
        if not given:
            return (None,) * 6
        with torch.no_grad():
            got = _rotary(given[0], given[1] if len(given) == 2 else None, positions, frequencies, *ctx.how, 1)
        got = iter(_once("rotary", tuple(got[:len(given)]), *given))
        return (*(None if t is None else next(got) for t in (dq, dk)), None, None, None, None)


def rotary(q, k, positions, frequencies, interleaved=False, magnitude=1.0):
    """Queries and keys turned by their positions, ``(q', k')``, with gradients; ``k`` may be None.  fp16, bf16 or fp32, any head size and strides.

    q and k are ``[batch, token, head, element]``, positions (int32 or int64) ``[batch, token]`` or ``[token]``.  The first ``part = 2 * len(frequencies)`` elements
    of a head are turned: pair i by ``positions * frequencies[i]`` radians (float64, as ``rotary_frequencies`` makes them) and times ``magnitude``; pair i is elements
    ``(i, i + part/2)``, or ``(2i, 2i + 1)`` where ``interleaved``.  The others stay.  There is no second derivative: asking for one raises."""
    out = _host().rotary(q, k, positions, frequencies, interleaved, magnitude)
    if out is not None:
        return out
    for name, t in (("q", q), ("k", k)):
        if t is None and name == "k":
            continue
        if not t.is_cuda or t.dtype not in _ROTARY_ELEMENT or t.dim() != 4:
            raise ValueError(f"{name} must be a [batch, token, head, element] GPU tensor of float16, bfloat16 or float32")
        if t.dtype != q.dtype or t.device != q.device or t.shape[:2] != q.shape[:2] or t.shape[3] != q.shape[3]:
            raise ValueError("q and k must have the same batch, tokens, head size, dtype and device")
    if frequencies.dtype != torch.float64 or frequencies.dim() != 1 or frequencies.device != q.device or frequencies.requires_grad:
        raise ValueError("frequencies must be a float64 vector on the device of q, without gradient")
    if not 1 <= frequencies.shape[0] <= min(q.shape[3], MAX_ROTARY_PART) // 2:
        raise ValueError(f"frequencies must be those of at most {MAX_ROTARY_PART} elements of a head")
    if positions.dtype not in (torch.int32, torch.int64) or positions.device != q.device:
        raise ValueError("positions must be int32 or int64 on the device of q")
    if tuple(positions.shape) not in ((q.shape[1],), tuple(q.shape[:2])):
        raise ValueError("positions must be [token] or [batch, token]")
    if not math.isfinite(magnitude):
        raise ValueError("magnitude must be finite")
    if positions.dim() == 1:
        positions = positions.expand(q.shape[0], -1)
    frequencies, magnitude = frequencies.contiguous(), float(magnitude)
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        return LEGORotary.apply(q, k, positions, frequencies, interleaved, magnitude)
    return tuple(_rotary(q, k, positions, frequencies, interleaved, magnitude, 0))
