"""Python mirror of the reference's MLX operator surface, backed by the C ABI.

Names, argument meaning and error behaviour follow
``overlays/executorch/backends/mlx/native_affine_ops.py`` (the torch custom
ops ``mlx::native_*`` that TriFuse's OLMoE export lowers onto MLX) plus the
runtime-level pieces of the OLMoE adapter (``olmoe_route``, the route sort,
``moe()``, the expert hook's GPU callable, T1 attention).  Every function
takes CUDA tensors and launches the sm_100a kernels of ``libtrifuse_b200.so``
on the current torch stream; there is no CPU path.  torch is used only to
allocate outputs and scratch.
"""
from __future__ import annotations

import ctypes as C
from array import array
from operator import index
from typing import NamedTuple

import torch
from torch import Tensor

from ._lib import (AffineWeight, CopyArray, DTYPE_BF16, DTYPE_E4M3, DTYPE_F16, DTYPE_F32, DTYPE_I8, MoeArgs, PagedKV,
                   PagedPlanDesc, PagedScales, PageTable, RouterWeight, TF_ERR_CAPACITY, check, lib)

_ACT = {torch.float16: DTYPE_F16, torch.bfloat16: DTYPE_BF16}


def _act(t: Tensor) -> int:
    if t.dtype not in _ACT:
        raise ValueError("activations must be float16 or bfloat16")
    return _ACT[t.dtype]


def _stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _ptr(t):
    return C.c_void_p(t.data_ptr()) if t is not None else None


def _cuda(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("trifuse_b200 ops take CUDA tensors (no CPU path)")


def _check_range(ids: Tensor, limit: int, message: str):
    """ids must lie in [0, limit): the kernels index with them unchecked
    (a host read of the extremes, one synchronization)."""
    if ids.numel() and (int(ids.min()) < 0 or int(ids.max()) >= limit):
        raise ValueError(message)


def _ws(nbytes: int, device) -> Tensor:
    return torch.empty(max(int(nbytes), 1), dtype=torch.uint8, device=device)


def validate_affine(q, scales, biases, group_size, bits, rank):
    """Same checks and messages as native_affine_ops.py:12-26."""
    if (type(bits) is not int or bits not in (4, 8)
            or type(group_size) is not int or group_size not in (32, 64, 128)):
        raise ValueError("Native affine requires bits4/8 and group32/64/128")
    if q.dtype != torch.uint32 or q.ndim != rank or rank not in (2, 3):
        raise ValueError("Native affine Q must be rank2/3 uint32")
    if (scales.dtype not in (torch.float16, torch.float32) or biases.dtype != scales.dtype
            or scales.shape != biases.shape or scales.ndim != rank
            or q.shape[:-1] != scales.shape[:-1]):
        raise ValueError("Native affine S/B shapes or floating dtypes differ")
    width = q.shape[-1] * (32 // bits)
    if (width % group_size or scales.shape[-1] * group_size != width
            or any(type(d) is not int or d <= 0 for d in q.shape)):
        raise ValueError("Native affine packed/group dimensions differ")
    if scales.dtype != torch.float16:
        raise NotImplementedError("this path consumes float16 scales/biases")
    return width


def affine_desc(q, scales, biases, group_size=64, bits=4) -> AffineWeight:
    width = validate_affine(q, scales, biases, group_size, bits, q.ndim)
    _cuda(q, scales, biases)
    for t in (q, scales, biases):
        if not t.is_contiguous():
            raise ValueError("Native affine Q/S/B must be contiguous")
    stacked = q.ndim == 3
    return AffineWeight(q.data_ptr(), scales.data_ptr(), biases.data_ptr(),
                        q.shape[0] if stacked else 0, q.shape[-2], width, group_size, bits)


def native_affine_qmm(x: Tensor, q: Tensor, scales: Tensor, biases: Tensor, group_size: int,
                      bits: int) -> Tensor:
    """``mlx::native_affine_qmm`` (native_affine_ops.py:39-52)."""
    w = affine_desc(q, scales, biases, group_size, bits)
    if q.ndim != 2:
        raise ValueError("Native affine Q must be rank2/3 uint32")
    if x.ndim < 1 or x.shape[-1] != w.in_features:
        raise ValueError("Native affine QMM input width/dtype differs")
    _cuda(x)
    x2 = x.contiguous().reshape(-1, w.in_features)
    y = torch.empty((*x.shape[:-1], w.out_features), dtype=x.dtype, device=x.device)
    check(lib().tf_affine_qmm(_ptr(x2), x2.shape[0], C.byref(w), _act(x), _ptr(y), _stream()))
    return y


def native_affine_gather_qmm(x: Tensor, q: Tensor, scales: Tensor, biases: Tensor, indices: Tensor,
                             group_size: int, bits: int, sorted_indices: bool = False) -> Tensor:
    """``mlx::native_affine_gather_qmm`` (native_affine_ops.py:55-74).

    Supports the reference's call forms (x[..., 1, H] broadcast against
    indices[...]): batch = broadcast(x.shape[:-2], indices.shape), output
    [*batch, 1, out]."""
    if q.ndim != 3:
        raise ValueError("Native affine Q must be rank2/3 uint32")
    w = affine_desc(q, scales, biases, group_size, bits)
    if indices.dtype not in (torch.int32, torch.int64):
        raise ValueError("Expert indices must be integers")
    if (x.ndim < 2 or x.shape[-1] != w.in_features or type(sorted_indices) is not bool):
        raise ValueError("Native affine expert input differs")
    if x.shape[-2] != 1:
        raise NotImplementedError("gather_qmm rows per expert call must be 1 (the adapter's forms)")
    _cuda(x, indices)
    batch = torch.broadcast_shapes(x.shape[:-2], indices.shape)
    xb = x.contiguous().reshape(-1, w.in_features)
    x_index = torch.arange(xb.shape[0], device=x.device, dtype=torch.int32).reshape(x.shape[:-2])
    x_index = x_index.expand(batch).reshape(-1).contiguous()
    idx = indices.to(torch.int32).expand(batch).reshape(-1).contiguous()
    _check_range(idx, w.experts, "expert index out of range")
    y = torch.empty((*batch, 1, w.out_features), dtype=x.dtype, device=x.device)
    check(lib().tf_affine_gather_qmm(_ptr(xb), xb.shape[0], 1, _ptr(x_index), _ptr(idx), idx.numel(),
                                     C.byref(w), int(sorted_indices), _act(x), _ptr(y), _stream()))
    return y


def native_affine_embedding(indices: Tensor, q: Tensor, scales: Tensor, biases: Tensor,
                            group_size: int, bits: int, out_dtype=torch.float16) -> Tensor:
    """``mlx::native_affine_embedding`` (native_affine_ops.py:77-93); output in
    the scales dtype (float16) unless out_dtype says otherwise."""
    if q.ndim != 2:
        raise ValueError("Native affine Q must be rank2/3 uint32")
    w = affine_desc(q, scales, biases, group_size, bits)
    if indices.dtype not in (torch.int32, torch.int64):
        raise ValueError("Embedding indices must be integers")
    _cuda(indices)
    ids = indices.to(torch.int64).reshape(-1).contiguous()
    if ids.numel() and (int(ids.min()) < 0 or int(ids.max()) >= w.out_features):
        raise ValueError("embedding index out of range")
    y = torch.empty((*indices.shape, w.in_features), dtype=out_dtype, device=indices.device)
    check(lib().tf_affine_embedding(_ptr(ids), ids.numel(), C.byref(w), _ACT[out_dtype], _ptr(y),
                                    _stream()))
    return y


def greedy_tokens(logits: Tensor) -> Tensor:
    """Greedy next tokens of fp32 logits [..., vocab]: argmax (lowest index on
    ties) where every logit of the row is finite, else -1 (int64); the
    reference's where(all(isfinite(logits)), argmax(logits), -1)
    (patches/executorch.patch:1350-1353)."""
    if logits.dtype != torch.float32:
        raise ValueError("greedy: logits must be float32")
    _cuda(logits)
    V = logits.shape[-1]
    lc = logits.contiguous().reshape(-1, V)
    out = torch.empty(lc.shape[0], dtype=torch.int64, device=logits.device)
    check(lib().tf_greedy_tokens(_ptr(lc), lc.shape[0], V, _ptr(out), _stream()))
    return out.reshape(logits.shape[:-1])


class TokenLogprobs(NamedTuple):
    """What token_logprobs reports of each row."""
    logprob: Tensor      # float32 [...]
    entropy: Tensor      # float32 [...], nats
    rank: Tensor         # int32 [...], 0 = argmax
    top_logprob: Tensor  # float32 [..., top]
    top_token: Tensor    # int64 [..., top]


def token_logprobs(logits: Tensor, tokens: Tensor, top: int = 0) -> TokenLogprobs:
    """Log probability of tokens [...] under logits [..., vocab] (float32,
    float16 or bfloat16), the distribution's entropy, the token's rank, and the
    ``top`` (at most 64) most probable tokens in order (ties: lower id first).

    A token outside the vocabulary (-1 for "none") gives NaN and rank -1, as
    does a row whose logits are NaN, +inf or all -inf."""
    if logits.dtype != torch.float32 and logits.dtype not in _ACT:
        raise ValueError("token_logprobs: logits must be float32, float16 or bfloat16")
    if logits.ndim < 1 or tokens.shape != logits.shape[:-1] or tokens.dtype != torch.int64:
        raise ValueError("token_logprobs: tokens are int64 with the shape of the logits' rows")
    if type(top) is not int:
        if not hasattr(type(top), "__index__"):
            raise ValueError("token_logprobs: top is an int")
        top = index(top)
    stream = _launch_stream(logits, tokens)
    shape, V = tokens.shape, logits.shape[-1]
    if logits.ndim != 2:
        logits = logits.reshape(-1, V)
    if logits.stride(1) != 1 or logits.stride(0) < V:
        logits = logits.contiguous()
    rows, k = logits.shape[0], max(top, 0)
    tokens = tokens.contiguous()
    logprob = torch.empty_like(tokens, dtype=torch.float32)
    entropy = torch.empty_like(logprob)
    rank = torch.empty_like(tokens, dtype=torch.int32)
    top_logprob = logprob.new_empty((*shape, k))
    top_token = tokens.new_empty((*shape, k))
    check(lib().tf_token_logprobs(logits.data_ptr(), logits.stride(0) if rows > 1 else V, rows, V,
                                  _ACT.get(logits.dtype, DTYPE_F32), tokens.data_ptr(), top, logprob.data_ptr(),
                                  entropy.data_ptr(), rank.data_ptr(), top_logprob.data_ptr(), top_token.data_ptr(),
                                  stream))
    return TokenLogprobs(logprob, entropy, rank, top_logprob, top_token)


class BeamChoice(NamedTuple):
    """The continuations that beam_select picks for each request, best first."""
    score: Tensor   # float32 [requests, count], -inf where there are fewer
    parent: Tensor  # int32 [requests, count], the beam that goes on; -1
    token: Tensor   # int64 [requests, count]; -1


def beam_select(logits: Tensor, scores: Tensor, count: int | None = None, finished: Tensor | None = None,
                end: int = -1) -> BeamChoice:
    """The ``count`` (default: as many as beams, at most 64) most probable
    continuations of each request over its beams and the vocabulary: logits
    [requests, beams, vocab] (float32, float16 or bfloat16), scores float32
    [requests, beams], the beams' log probabilities so far (-inf: no beam).

    A continuation's score is the beam's plus the token's log probability;
    equal ones in order of the beam, then of the token.  A beam marked in
    ``finished`` (bool [requests, beams]) goes on as it is, with the token
    ``end``.  Beams whose logits are no distribution, and tokens at -inf, have
    no continuation."""
    if logits.dtype != torch.float32 and logits.dtype not in _ACT:
        raise ValueError("beam_select: logits must be float32, float16 or bfloat16")
    if logits.ndim != 3 or scores.shape != logits.shape[:2] or scores.dtype != torch.float32:
        raise ValueError("beam_select: logits are [requests, beams, vocab], scores float32 [requests, beams]")
    if finished is not None and (finished.shape != scores.shape or finished.dtype != torch.bool):
        raise ValueError("beam_select: finished is bool [requests, beams]")
    R, beams, V = logits.shape
    count = beams if count is None else index(count)
    end = index(end)
    if not 1 <= count <= 64 or not -(1 << 63) <= end < 1 << 63:  # would wrap on the way to C
        raise ValueError("beam_select: count is from 1 to 64, end fits 64 bits")
    stream = _launch_stream(logits, scores, finished)
    step = V  # from row to row
    if not logits.is_contiguous():
        stride = logits.stride()
        step = stride[1] if beams > 1 else stride[0] if R > 1 else V
        if (V > 1 and stride[2] != 1) or step < V or (R > 1 and stride[0] != beams * step):
            logits, step = logits.contiguous(), V
    scores = scores.contiguous()
    if finished is not None:
        finished = finished.contiguous()
    # What tf_beam_select_workspace_size gives; checked by the call.
    ws = torch.empty(max(R * beams * (16 + 8 * min(count, V)), 1), dtype=torch.uint8, device=logits.device)
    score = torch.empty_like(scores) if count == beams else scores.new_empty((R, count))
    parent = torch.empty_like(score, dtype=torch.int32)
    token = torch.empty_like(score, dtype=torch.int64)
    check(lib().tf_beam_select(logits.data_ptr(), step, R, beams, V, _ACT.get(logits.dtype, DTYPE_F32),
                               scores.data_ptr(), None if finished is None else finished.data_ptr(), end, count,
                               score.data_ptr(), parent.data_ptr(), token.data_ptr(), ws.data_ptr(), ws.numel(),
                               stream))
    return BeamChoice(score, parent, token)


def native_olmoe_softmax(x: Tensor) -> Tensor:
    """``mlx::native_olmoe_softmax`` (native_affine_ops.py:128-138): fp32
    softmax over the last axis, rounded to the storage dtype."""
    _cuda(x)
    E = x.shape[-1]
    xc = x.contiguous()
    p = torch.empty_like(xc)
    check(lib().tf_olmoe_softmax(_ptr(xc), xc.numel() // E, E, _act(x), _ptr(p), _stream()))
    return p


def native_olmoe_topk_indices(x: Tensor, k: int) -> Tensor:
    """``mlx::native_olmoe_topk_indices`` (native_affine_ops.py:141-153):
    stable descending rank (ties to lower id, NaN last), first k, int32."""
    if type(k) is not int or not 0 < k <= x.shape[-1]:
        raise ValueError("Invalid OLMoE top-k")
    _cuda(x)
    E = x.shape[-1]
    xc = x.contiguous()
    out = torch.empty((*x.shape[:-1], k), dtype=torch.int32, device=x.device)
    check(lib().tf_olmoe_topk_indices(_ptr(xc), xc.numel() // E, E, k, _act(x), _ptr(out), _stream()))
    return out


def native_take_along_last(x: Tensor, indices: Tensor) -> Tensor:
    """``mlx::native_take_along_last`` (native_affine_ops.py:115-125)."""
    if (x.ndim < 1 or x.shape[:-1] != indices.shape[:-1]
            or indices.dtype not in (torch.int32, torch.int64)):
        raise ValueError("Native take requires matching leading dimensions and integer indices")
    _cuda(x, indices)
    W, K = x.shape[-1], indices.shape[-1]
    xc = x.contiguous()
    ic = indices.to(torch.int32).contiguous()
    out = torch.empty(indices.shape, dtype=x.dtype, device=x.device)
    check(lib().tf_take_along_last(_ptr(xc), xc.numel() // W, W, _ptr(ic), K, _act(x), _ptr(out),
                                   _stream()))
    return out


def olmoe_route(logits: Tensor, k: int):
    """``olmoe_route`` (MLXOLMoERouter.h:86-120): (indices int32, gates act)."""
    if type(k) is not int or not 0 < k <= logits.shape[-1]:
        raise ValueError("OLMoE router geometry differs")
    _cuda(logits)
    E = logits.shape[-1]
    lc = logits.contiguous()
    idx = torch.empty((*logits.shape[:-1], k), dtype=torch.int32, device=logits.device)
    gates = torch.empty((*logits.shape[:-1], k), dtype=logits.dtype, device=logits.device)
    check(lib().tf_olmoe_route(_ptr(lc), lc.numel() // E, E, k, _act(logits), _ptr(idx), _ptr(gates),
                               _stream()))
    return idx, gates


def router_desc(router) -> RouterWeight:
    """A dense act weight [E,H] or an affine (q, scales, biases) triple."""
    if isinstance(router, Tensor):
        _cuda(router)
        return RouterWeight(router.contiguous().data_ptr(), AffineWeight())
    q, s, b = router
    return RouterWeight(None, affine_desc(q, s, b))


def olmoe_router(x: Tensor, router, k: int, experts: int | None = None):
    """Router GEMV + route (MLXNativeGraniteMoEPrefill.h:631-632):
    returns (logits, indices, gates)."""
    _cuda(x)
    H = x.shape[-1]
    E = router.shape[0] if isinstance(router, Tensor) else router[0].shape[0]
    rw = router_desc(router)
    xc = x.contiguous().reshape(-1, H)
    T = xc.shape[0]
    logits = torch.empty((T, E), dtype=x.dtype, device=x.device)
    idx = torch.empty((T, k), dtype=torch.int32, device=x.device)
    gates = torch.empty((T, k), dtype=x.dtype, device=x.device)
    check(lib().tf_olmoe_router(_ptr(xc), T, H, C.byref(rw), E, k, _act(x), _ptr(logits), _ptr(idx),
                                _ptr(gates), _stream()))
    return logits, idx, gates


def moe_route_sort(indices: Tensor, experts: int):
    """Stable grouping of routes by expert (MLXNativeGraniteMoEPrefill.h:
    666-684): (order, inverse, offsets[E+1]), int32."""
    _cuda(indices)
    idx = indices.to(torch.int32).contiguous()
    _check_range(idx, experts, "expert index out of range")
    T = idx.shape[0] if idx.ndim > 1 else idx.numel()
    K = idx.shape[-1] if idx.ndim > 1 else 1
    n = idx.numel()
    order = torch.empty(n, dtype=torch.int32, device=idx.device)
    inverse = torch.empty(n, dtype=torch.int32, device=idx.device)
    offsets = torch.empty(experts + 1, dtype=torch.int32, device=idx.device)
    nb = C.c_size_t()
    check(lib().tf_moe_route_sort_workspace_size(T, K, experts, C.byref(nb)))
    ws = _ws(nb.value, idx.device)
    check(lib().tf_moe_route_sort(_ptr(idx), T, K, experts, _ptr(order), _ptr(inverse), _ptr(offsets),
                                  _ptr(ws), nb.value, _stream()))
    return order, inverse, offsets


def moe_combine(y_sorted: Tensor, inverse: Tensor, gates: Tensor, residual: Tensor) -> Tensor:
    """Top-k combine + residual (MLXNativeGraniteMoEPrefill.h:688-695): rows of
    y_sorted are in route-sort order, inverse maps each route t*k+j to its row."""
    _cuda(y_sorted, inverse, gates, residual)
    T, K = gates.shape
    H = residual.shape[-1]
    if y_sorted.shape != (T * K, H) or inverse.numel() != T * K or residual.shape != (T, H):
        raise ValueError("moe_combine: shape mismatch")
    if not (y_sorted.dtype == gates.dtype == residual.dtype):
        raise ValueError("moe_combine: y, gates and residual share the activation dtype")
    out = torch.empty_like(residual)
    check(lib().tf_moe_combine(_ptr(y_sorted.contiguous()), _ptr(inverse.to(torch.int32).contiguous()),
                               _ptr(gates.contiguous()), _ptr(residual.contiguous()), T, K, H,
                               _act(residual), _ptr(out), _stream()))
    return out


def moe_args(x, residual, out, router, gate, up, down, top_k, logits=None, indices=None, gates=None):
    H = x.shape[-1]
    T = x.numel() // H
    g = affine_desc(*gate)
    a = MoeArgs()
    a.x, a.residual, a.out = x.data_ptr(), residual.data_ptr(), out.data_ptr()
    a.tokens, a.hidden, a.intermediate = T, H, g.out_features
    a.experts, a.top_k, a.act = g.experts, top_k, _act(x)
    a.router = router_desc(router)
    a.gate_proj, a.up_proj, a.down_proj = g, affine_desc(*up), affine_desc(*down)
    a.logits = logits.data_ptr() if logits is not None else None
    a.indices = indices.data_ptr() if indices is not None else None
    a.gates = gates.data_ptr() if gates is not None else None
    return a


def moe(x: Tensor, residual: Tensor, router, gate, up, down, top_k: int, return_aux=False):
    """One OLMoE sparse-MoE block (``moe()``, MLXNativeGraniteMoEPrefill.h:627-702):
    residual + sum_k gate_k * down(silu(gate(x)) * up(x))."""
    _cuda(x, residual)
    if x.shape != residual.shape or x.dtype != residual.dtype:
        raise ValueError("moe: x and residual must match")
    x = x.contiguous()
    residual = residual.contiguous()
    H = x.shape[-1]
    T = x.numel() // H
    E = gate[0].shape[0]
    out = torch.empty_like(x)
    logits = torch.empty((T, E), dtype=x.dtype, device=x.device) if return_aux else None
    idx = torch.empty((T, top_k), dtype=torch.int32, device=x.device) if return_aux else None
    gates = torch.empty((T, top_k), dtype=x.dtype, device=x.device) if return_aux else None
    a = moe_args(x, residual, out, router, gate, up, down, top_k, logits, idx, gates)
    nb = C.c_size_t()
    check(lib().tf_moe_workspace_size(C.byref(a), C.byref(nb)))
    ws = _ws(nb.value, x.device)
    check(lib().tf_moe_forward(C.byref(a), _ptr(ws), nb.value, _stream()))
    if return_aux:
        return out, dict(logits=logits, indices=idx, gates=gates)
    return out


def expert_gpu(x: Tensor, token_indices: Tensor, expert_ids: Tensor, experts_sorted: bool, gate, up,
               down):
    """The expert hook's ``GPUCallable`` (MLXMoEExpertHook.h:25-32): returns
    (expert-sorted output [N, H], inverse [N])."""
    if (token_indices.ndim != 1 or expert_ids.ndim != 1 or token_indices.shape != expert_ids.shape
            or token_indices.dtype not in (torch.int32,) or expert_ids.dtype not in (torch.int32,)):
        raise ValueError("expert hook route arrays must be parallel integer vectors")
    _cuda(x, token_indices, expert_ids)
    H = x.shape[-1]
    xc = x.contiguous().reshape(-1, H)
    g, u, d = affine_desc(*gate), affine_desc(*up), affine_desc(*down)
    _check_range(expert_ids, g.experts, "expert index out of range")
    _check_range(token_indices, xc.shape[0], "token index out of range")
    n = token_indices.numel()
    out = torch.empty((n, H), dtype=x.dtype, device=x.device)
    inverse = torch.empty(n, dtype=torch.int32, device=x.device)
    nb = C.c_size_t()
    check(lib().tf_moe_expert_workspace_size(n, xc.shape[0], H, g.out_features, g.experts, _act(x),
                                             C.byref(nb)))
    ws = _ws(nb.value, x.device)
    check(lib().tf_moe_expert_gpu(_ptr(xc), xc.shape[0], H, _ptr(token_indices), _ptr(expert_ids), n,
                                  int(experts_sorted), g.out_features, g.experts, C.byref(g), C.byref(u),
                                  C.byref(d), _act(x), _ptr(out), _ptr(inverse), _ptr(ws), nb.value,
                                  _stream()))
    return out, inverse


def expert_gpu_ordered(x: Tensor, token_indices: Tensor, expert_ids: Tensor, gate, up, down,
                       check_ranges: bool = True) -> Tensor:
    """The expert hook's computation with the output rows in the routes' own
    order (row i for route i); no inverse permutation.  check_ranges=False
    skips the host-side index checks (one device-to-host read each) for
    callers whose indices are valid by construction."""
    if (token_indices.ndim != 1 or expert_ids.ndim != 1 or token_indices.shape != expert_ids.shape
            or token_indices.dtype != torch.int32 or expert_ids.dtype != torch.int32):
        raise ValueError("expert hook route arrays must be parallel integer vectors")
    _cuda(x, token_indices, expert_ids)
    H = x.shape[-1]
    xc = x.contiguous().reshape(-1, H)
    g, u, d = affine_desc(*gate), affine_desc(*up), affine_desc(*down)
    if check_ranges:
        _check_range(expert_ids, g.experts, "expert index out of range")
        _check_range(token_indices, xc.shape[0], "token index out of range")
    n = token_indices.numel()
    out = torch.empty((n, H), dtype=x.dtype, device=x.device)
    nb = C.c_size_t()
    check(lib().tf_moe_expert_workspace_size(n, xc.shape[0], H, g.out_features, g.experts, _act(x),
                                             C.byref(nb)))
    ws = _ws(nb.value, x.device)
    check(lib().tf_moe_expert_gpu_ordered(_ptr(xc), xc.shape[0], H, _ptr(token_indices), _ptr(expert_ids), n,
                                          g.out_features, g.experts, C.byref(g), C.byref(u), C.byref(d),
                                          _act(x), _ptr(out), _ptr(ws), nb.value, _stream()))
    return out


def gather_rows(x: Tensor, index: Tensor, div: int = 1) -> Tensor:
    """y[i] = x[index[i] // div] (rows of the activation dtype); index int32
    on the device, in range by the caller's construction."""
    _cuda(x, index)
    if index.dtype != torch.int32 or index.ndim != 1:
        raise ValueError("gather_rows: int32 index vector")
    H = x.shape[-1]
    xc = x.contiguous().reshape(-1, H)
    n = index.numel()
    y = torch.empty((n, H), dtype=x.dtype, device=x.device)
    check(lib().tf_gather_rows(_ptr(xc), xc.shape[0], H, _ptr(index), int(div), n, _act(x), _ptr(y), _stream()))
    return y


def rms_norm(x: Tensor, weight: Tensor, eps: float) -> Tensor:
    """``fast::rms_norm`` as used by the adapter (MLXNativeGraniteMoEPrefill.h:434)."""
    _cuda(x, weight)
    W = x.shape[-1]
    xc = x.contiguous()
    y = torch.empty_like(xc)
    check(lib().tf_rms_norm(_ptr(xc), xc.numel() // W, W, _ptr(weight.contiguous()), eps, _act(x), _ptr(y),
                            _stream()))
    return y


def attention_decode(qkv: Tensor, q_norm: Tensor, k_norm: Tensor, positions: Tensor, k_cache: Tensor,
                     v_cache: Tensor, eps: float, rope_theta: float, scale: float | None = None,
                     max_length: int | None = None) -> Tensor:
    """T1 attention for a batch of requests (MLXNativeGraniteMoEPrefill.h:446-483):
    q/k full-width RMSNorm, RoPE, KV append at positions[b], SDPA.
    k_cache/v_cache: float16 [batch, heads, capacity, head_dim] (updated)."""
    _cuda(qkv, q_norm, k_norm, positions, k_cache, v_cache)
    B, heads, cap, D = k_cache.shape
    if qkv.shape != (B, 3 * heads * D) or v_cache.shape != k_cache.shape:
        raise ValueError("attention: qkv/cache geometry differs")
    if k_cache.dtype != torch.float16 or v_cache.dtype != torch.float16:
        raise ValueError("ordered full-history FP16 KV required")
    scale = D ** -0.5 if scale is None else scale
    max_length = cap if max_length is None else max_length
    pos = positions.to(torch.int32).contiguous()
    out = torch.empty((B, heads * D), dtype=qkv.dtype, device=qkv.device)
    nb = C.c_size_t()
    check(lib().tf_attention_decode_workspace_size(B, heads, cap, C.byref(nb)))
    ws = _ws(nb.value, qkv.device)
    check(lib().tf_attention_decode(_ptr(qkv.contiguous()), B, heads, D, _ptr(q_norm), _ptr(k_norm), eps,
                                    rope_theta, _ptr(pos), max_length, _ptr(k_cache), _ptr(v_cache), cap,
                                    scale, _act(qkv), _ptr(out), _ptr(ws), nb.value, _stream()))
    return out


# ---------------------------------------------------------------------------
# paged key/value cache


SCALE_TOKENS = 16  # tokens of a page and head that share a scale in an 8-bit cache
_CODES = {torch.int8: DTYPE_I8, torch.float8_e4m3fn: DTYPE_E4M3}


def _paged_kv(k_pages: Tensor, v_pages: Tensor, types=_ACT) -> PagedKV:
    """Descriptor of [pages, kv_heads, page_size, head_dim] caches; only the
    first dimension may have a stride of its own."""
    shape, dtype, stride = k_pages.shape, k_pages.dtype, k_pages.stride()
    if len(shape) != 4 or shape != v_pages.shape or dtype != v_pages.dtype:
        raise ValueError("paged: k_pages and v_pages are [pages, kv_heads, page_size, head_dim] of one dtype")
    if dtype not in types:
        if types is _CODES:
            raise ValueError("paged: a cache with scales must be int8 or float8_e4m3fn")
        if dtype in _CODES:
            raise ValueError("paged: an 8-bit cache needs k_scales and v_scales")
        raise ValueError("paged: the cache must be float16 or bfloat16")
    pages, heads, size, D = shape
    other = v_pages.stride()
    if heads == 1 or pages == 1:  # the stride of a dimension of one is of no meaning
        stride, other = ((t[0] if pages > 1 else heads * size * D, t[1] if heads > 1 else size * D, t[2], t[3])
                         for t in (stride, other))
    step = stride[0]
    if stride != (step, size * D, D, 1) or stride != other:
        raise ValueError("paged: a page must be contiguous, and k_pages and v_pages laid out alike")
    return PagedKV(k_pages.data_ptr(), v_pages.data_ptr(), pages, step, heads, size, D, types[dtype])


def _paged_scales(k_scales: Tensor | None, v_scales: Tensor | None, kv: PagedKV) -> PagedScales:
    """Descriptor of the scales [pages, kv_heads, page_size / 16] of an 8-bit
    cache; only the first dimension may have a stride of its own."""
    if k_scales is None or v_scales is None:
        raise ValueError("paged: k_scales and v_scales go together")
    pages, heads, blocks = kv.pages, kv.kv_heads, kv.page_size // SCALE_TOKENS
    if (k_scales.shape != (pages, heads, blocks) or v_scales.shape != (pages, heads, blocks)
            or k_scales.dtype != torch.float32 or v_scales.dtype != torch.float32):
        raise ValueError("paged: scales are float32 [pages, kv_heads, page_size / 16]")
    stride, other = k_scales.stride(), v_scales.stride()
    if pages == 1 or heads == 1 or blocks == 1:  # the stride of a dimension of one is of no meaning
        stride, other = ((t[0] if pages > 1 else heads * blocks, t[1] if heads > 1 else blocks, t[2] if blocks > 1 else 1)
                         for t in (stride, other))
    if stride != other or stride[1] != blocks or stride[2] != 1:
        raise ValueError("paged: a page's scales must be contiguous, and k_scales and v_scales laid out alike")
    return PagedScales(k_scales.data_ptr(), v_scales.data_ptr(), stride[0])


def _page_table(page_table: Tensor) -> PageTable:
    """Descriptor of a page table; keep both until the launch."""
    shape, stride = page_table.shape, page_table.stride()
    if len(shape) != 2 or page_table.dtype != torch.int32 or (shape[1] > 1 and stride[1] != 1):
        raise ValueError("paged: the page table is int32 [requests, pages] with contiguous rows")
    requests, columns = shape
    if stride[0] >= columns:
        return PageTable(page_table.data_ptr(), stride[0], requests, columns)
    if requests > 1:  # rows that share memory (an expanded row) are laid out apart
        page_table = page_table.clone(memory_format=torch.contiguous_format)
    desc = PageTable(page_table.data_ptr(), columns, requests, columns)  # the stride of one row is of no meaning
    desc.tensor = page_table
    return desc


def _launch_stream(first: Tensor, *others) -> int:
    """The current device's current stream (its handle); every tensor must live on that device."""
    dev = first.get_device()
    for t in others:
        if t is not None and t.get_device() != dev:
            _cuda(first, *others)
            raise ValueError("tensors must be on one CUDA device")
    _cuda(first)
    if dev != torch._C._cuda_getDevice():
        raise ValueError("tensors must be on the current CUDA device")
    return torch._C._cuda_getCurrentRawStream(dev)


def _rows16(t: Tensor, width: int) -> Tensor:
    """t, or a copy of it where its rows (of `width` values) cannot be read 16 bytes at a time."""
    step = t.stride(0)
    if step < width or step % 8 or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _norm_weight(w: Tensor, n: int):
    """A norm's n weights (or a copy of them where they start off 16 bytes) and their address."""
    if w.dtype != torch.float16 or w.shape != (n,) or not w.is_contiguous():
        raise ValueError("paged_append: norm weights are contiguous float16 over the full q and k widths")
    at = w.data_ptr()
    if at % 16:
        w = w.clone()
        at = w.data_ptr()
    return w, at


def paged_append(qkv: Tensor, k_pages: Tensor, v_pages: Tensor, page_table: Tensor, positions: Tensor,
                 requests: Tensor, heads: int, q_norm: Tensor | None = None, k_norm: Tensor | None = None,
                 eps: float = 1e-5, rope_theta: float | None = None, out: Tensor | None = None,
                 k_scales: Tensor | None = None, v_scales: Tensor | None = None) -> Tensor:
    """New tokens into a paged cache: q and k RMS-normalised over their full
    widths (when norms are given) and rotated by halves at ``positions`` (when
    ``rope_theta`` is given), k and v written to the pages (updated in place),
    q returned as [rows, heads, head_dim].

    qkv: [rows, (heads + 2 kv_heads) * head_dim] rows q | k | v; positions and
    requests: int32 [rows] on the device; page_table: int32 [requests, pages].
    A row whose slot the table does not have is not stored.

    An 8-bit cache (int8 or float8_e4m3fn pages) comes with k_scales and
    v_scales, float32 [pages, kv_heads, page_size / 16], updated in place: a
    block of 16 tokens and a head have the scale of their largest magnitude,
    which becomes the code 127 (int8) or 448.  Where new tokens raise it, the
    block's earlier codes are rounded anew.  Rows of a request whose tokens
    share a block are adjacent, in rising order."""
    stream = _launch_stream(qkv, k_pages, v_pages, page_table, positions, requests, q_norm, k_norm, out, k_scales,
                            v_scales)
    coded = k_scales is not None or v_scales is not None
    kv = _paged_kv(k_pages, v_pages, _CODES if coded else _ACT)
    D, kv_heads = kv.head_dim, kv.kv_heads
    width = (heads + 2 * kv_heads) * D
    if qkv.ndim != 2 or qkv.shape[1] != width:
        raise ValueError("paged_append: qkv is [rows, (heads + 2 kv_heads) * head_dim]")
    qkv = _rows16(qkv if qkv.stride(1) == 1 else qkv.contiguous(), width)
    rows = qkv.shape[0]
    i32 = torch.int32
    if (positions.dtype != i32 or requests.dtype != i32 or not positions.shape == requests.shape == (rows,)
            or not positions.is_contiguous() or not requests.is_contiguous()):
        raise ValueError("paged_append: positions and requests are contiguous int32 [rows]")
    qn = kn = None
    if q_norm is not None:
        q_norm, qn = _norm_weight(q_norm, heads * D)
    if k_norm is not None:
        k_norm, kn = _norm_weight(k_norm, kv_heads * D)
    q = out
    if out is None:
        q = qkv.new_empty((rows, heads, D))
    elif out.shape != (rows, heads, D) or out.dtype != qkv.dtype or not out.is_contiguous():
        raise ValueError("paged_append: out is a contiguous [rows, heads, head_dim] of qkv's dtype")
    elif out.data_ptr() % 16:  # the kernel cannot store there: copied over
        q = torch.empty_like(out)
    args = (qkv.data_ptr(), qkv.stride(0) if rows > 1 else width, rows, heads, _act(qkv), qn, kn, eps,
            rope_theta or 0.0, positions.data_ptr(), requests.data_ptr(), _page_table(page_table), kv)
    if coded:
        check(lib().tf_paged_append_8bit(*args, _paged_scales(k_scales, v_scales, kv), q.data_ptr(), stream))
    else:
        check(lib().tf_paged_append(*args, q.data_ptr(), stream))
    return q if out is None or out is q else out.copy_(q)


class PagedPlan:
    """How one paged attention call is divided over the GPU, from the lengths
    and the geometry alone: made once per step, used in every layer.

    new_lengths[i] query rows and kv_lengths[i] cached tokens (the new ones
    included) of request i, as sequences of ints.  ``positions`` and
    ``requests`` are the rows' int32 device vectors for ``paged_append``,
    ordered after the plan's upload on the stream that is current when they are
    asked for.  The plan holds the calls' workspace, so calls that may run at
    the same time (on several streams) need plans of their own."""

    def __init__(self, new_lengths, kv_lengths, heads: int, kv_heads: int, head_dim: int, page_size: int,
                 device=None):
        n = len(new_lengths)
        if len(kv_lengths) != n:
            raise ValueError("paged plan: new_lengths and kv_lengths differ in length")
        new_lengths, kv_lengths = [index(x) for x in new_lengths], [index(x) for x in kv_lengths]
        if any(not -(1 << 31) <= x < 1 << 31 for x in new_lengths + kv_lengths):  # would wrap on the way to C
            raise ValueError("paged plan: a length does not fit 32 bits")
        if torch.cuda.is_current_stream_capturing():  # a replay would read host memory that is long reused
            raise RuntimeError("paged plan: made while the stream captures a graph; make it before the capture")
        new, kv = (C.c_int32 * n)(*new_lengths), (C.c_int32 * n)(*kv_lengths)
        self.desc = d = PagedPlanDesc()
        # At most 4 MB before the planner has checked what it is to plan.
        guess = 65536 + min(64 * n * max(kv_heads, 1) + 16 * max(sum(new_lengths), 0), 1 << 22)
        while True:  # a second time when the table outgrows the guess
            host = torch.empty(guess, dtype=torch.uint8, pin_memory=True)
            status = lib().tf_paged_plan_make(new, kv, n, heads, kv_heads, head_dim, page_size, d, host.data_ptr(),
                                              guess)
            if status != TF_ERR_CAPACITY:
                break
            guess = d.table_bytes
        check(status)
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        self.table = host[:d.table_bytes].to(device, non_blocking=True)
        self.workspace = torch.empty(max(d.workspace_bytes, 1), dtype=torch.uint8, device=device)
        stream = torch.cuda.current_stream(device)
        self.made_on = stream.cuda_stream
        self.device_index = self.table.get_device()
        self._ready = stream.record_event()
        self.shape = (d.rows, heads, head_dim)  # of q
        self.rows = d.rows
        self.table_ptr, self.workspace_ptr = self.table.data_ptr(), self.workspace.data_ptr()
        self.workspace_bytes, self.widened_bytes = d.workspace_bytes, d.widened_bytes
        at, size = d.positions_offset, 4 * d.rows
        self._positions = self.table[at:at + size].view(torch.int32)
        at = d.requests_offset
        self._requests = self.table[at:at + size].view(torch.int32)

    def _here(self, vector: Tensor) -> Tensor:
        handle = torch._C._cuda_getCurrentRawStream(self.device_index)
        if handle != self.made_on:
            self.order(handle)
        return vector

    @property
    def positions(self) -> Tensor:
        return self._here(self._positions)

    @property
    def requests(self) -> Tensor:
        return self._here(self._requests)

    def order(self, handle: int):
        """Orders the plan's upload before work on another stream (the current
        one, of this handle) and keeps its memory until that work is done.  A
        capturing stream cannot wait for an event from outside; a graph's first
        replay comes after the synchronization that opens its capture, and its
        owner keeps the plan."""
        if handle != self.made_on and not torch.cuda.is_current_stream_capturing():
            stream = torch.cuda.current_stream(self.device_index)
            stream.wait_event(self._ready)
            self.table.record_stream(stream)
            self.workspace.record_stream(stream)


def paged_attention(q: Tensor, k_pages: Tensor, v_pages: Tensor, page_table: Tensor, plan: PagedPlan,
                    scale: float | None = None, out: Tensor | None = None, k_scales: Tensor | None = None,
                    v_scales: Tensor | None = None) -> Tensor:
    """Attention of every request's new tokens over its pages: row i of a
    request attends keys 0 .. kv_length - new_length + i; query heads share
    key heads in groups.  q: [rows, heads, head_dim] (rows may be strided);
    returns [rows, heads, head_dim].  Rows that attend nothing give zeros.

    An 8-bit cache (int8 or float8_e4m3fn pages) comes with the k_scales and
    v_scales that ``paged_append`` keeps; a plan serves either kind of cache."""
    stream = _launch_stream(q, k_pages, v_pages, page_table, plan.table, out, k_scales, v_scales)
    shape = plan.shape
    if q.shape != shape:
        raise ValueError("paged_attention: q is [rows, heads, head_dim] of the plan")
    rows, heads, D = shape
    width = heads * D
    q = _rows16(q if q.stride()[1:] == (D, 1) else q.contiguous(), width)
    o = out
    if out is None:
        o = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != shape or out.dtype != q.dtype or not out.is_contiguous():
        raise ValueError("paged_attention: out is a contiguous [rows, heads, head_dim] of q's dtype")
    elif out.data_ptr() % 32:  # the kernel cannot store there: copied over
        o = torch.empty_like(out)
    if stream != plan.made_on:
        plan.order(stream)
    q_stride = q.stride(0) if rows > 1 else width
    scale = D ** -0.5 if scale is None else scale
    if k_scales is None and v_scales is None:
        check(lib().tf_paged_attention(q.data_ptr(), q_stride, _page_table(page_table), _paged_kv(k_pages, v_pages),
                                       plan.desc, plan.table_ptr, scale, _act(q), o.data_ptr(), plan.workspace_ptr,
                                       plan.workspace_bytes, stream))
    else:
        kv = _paged_kv(k_pages, v_pages, _CODES)
        ws, nbytes = plan.workspace_ptr, plan.workspace_bytes
        if plan.widened_bytes:  # of this call alone: other steps' plans need not hold it
            nbytes += plan.widened_bytes
            widened = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
            ws = widened.data_ptr()
        check(lib().tf_paged_attention_8bit(q.data_ptr(), q_stride, _page_table(page_table), kv,
                                            _paged_scales(k_scales, v_scales, kv), plan.desc, plan.table_ptr, scale,
                                            _act(q), o.data_ptr(), ws, nbytes, stream))
    return o if out is None or out is o else out.copy_(o)


def paged_copy(arrays, src, dst):
    """Page dst[i] becomes page src[i] in every layer of every array (a cache's
    keys, values and scales: up to 8 tensors [layers, pages, ...] with
    contiguous pages, updated in place).  src and dst are sequences of ints on
    the host.  A page may be written once, and not be read as well."""
    arrays = list(arrays)
    if not arrays:
        raise ValueError("paged_copy: no arrays")
    stream = _launch_stream(*arrays)
    layers, pages = arrays[0].shape[:2] if arrays[0].ndim > 1 else (0, 0)
    descs = []
    for t in arrays:
        shape, stride, size = t.shape, t.stride(), t.element_size()
        if len(shape) < 3 or shape[0] != layers or shape[1] != pages:
            raise ValueError("paged_copy: arrays are [layers, pages, ...] with the same layers and pages")
        if t.is_contiguous():
            n = t.numel() // max(layers * pages, 1)  # values of a page
        else:
            n = 1
            for i in range(len(shape) - 1, 1, -1):  # the stride of a dimension of one is of no meaning
                if shape[i] != 1 and stride[i] != n:
                    raise ValueError("paged_copy: a page must be contiguous")
                n *= shape[i]
            if (pages > 1 and stride[1] < n) or (layers > 1 and stride[0] == 0):
                raise ValueError("paged_copy: pages share memory")
        descs.append(CopyArray(t.data_ptr(), stride[0] * size if layers > 1 else 0,
                               (stride[1] if pages > 1 else n) * size, n * size))
    try:
        src, dst = array("i", src), array("i", dst)
    except OverflowError:
        raise ValueError("paged_copy: a page does not fit 32 bits") from None
    if len(src) != len(dst):
        raise ValueError("paged_copy: src and dst differ in length")
    check(lib().tf_paged_copy((CopyArray * len(descs))(*descs), len(descs), layers, pages, src.buffer_info()[0],
                              dst.buffer_info()[0], len(src), stream))


def set_qmm_path(path: int):
    """0 = automatic, 1 = CUDA-core GEMV only, 2 = tensor cores when eligible."""
    check(lib().tf_set_qmm_path(int(path)))


def device_error(clear: bool = True) -> int:
    """First error code recorded by a device-side bounded wait (0 = none)."""
    return lib().tf_device_error(int(clear))
