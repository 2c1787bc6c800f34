"""Tensor-level wrappers of the C ABI. Every op runs the HIP kernels; none has a CPU path.

All tensors must live on one ROCm device; outputs are allocated with torch (caching
allocator, so the ops are safe to capture in a HIP graph) and every launch goes to
torch.cuda.current_stream().
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from mtp_amd import _lib
from mtp_amd.weights import Int8Experts, MoeExperts

PATHS = {"auto": _lib.PATH_AUTO, "decode": _lib.PATH_DECODE, "prefill": _lib.PATH_PREFILL}
DECODE_BLOCK_M = 16
PREFILL_BLOCK_M = 128
AUTO_PREFILL_SLOTS = 2560  # routed slots (T * top_k) from which "auto" runs the prefill path
OUT_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def _stream() -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _require_gpu(*tensors: torch.Tensor | None) -> None:
    dev = None
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError("the W4A16 MoE kernels need ROCm device tensors; got a CPU tensor")
        if not t.is_contiguous():
            raise ValueError("tensors passed to the W4A16 MoE kernels must be contiguous")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise ValueError(f"tensors on different devices: {dev} and {t.device}")


def _require_experts_on(device: torch.device, *sets: MoeExperts | None) -> None:
    """Expert sets are validated by MoeExperts.validate (contiguous stacks or slot-pool views);
    here only their device is checked against the activations'."""
    for ex in sets:
        if ex is not None and ex.device != device:
            raise ValueError(f"expert weights on {ex.device}, activations on {device}")


def _workspace(workspace: torch.Tensor | None, need: int, device: torch.device) -> torch.Tensor:
    """The caller's workspace when it is a contiguous tensor on ``device`` of at least ``need``
    bytes; a smaller one is replaced by a new allocation."""
    if workspace is not None:
        if not workspace.is_cuda or workspace.device != device or not workspace.is_contiguous():
            raise ValueError(f"workspace must be a contiguous tensor on {device}")
        if _nbytes(workspace) >= need:
            return workspace
    return torch.empty(max(need, 1), dtype=torch.uint8, device=device)


def _nbytes(t: torch.Tensor) -> int:
    return t.numel() * t.element_size()


def _path(path: str | int) -> int:
    if isinstance(path, int):
        return path
    try:
        return PATHS[path]
    except KeyError as exc:
        raise ValueError(f"path must be one of {sorted(PATHS)}") from exc


def _bf16_matrix(x: torch.Tensor, name: str, cols: int | None = None) -> None:
    if x.dtype != torch.bfloat16:
        raise TypeError(f"{name} must be bfloat16, got {x.dtype}")
    if x.ndim != 2:
        raise ValueError(f"{name} must be 2D, got {tuple(x.shape)}")
    if cols is not None and x.shape[1] != cols:
        raise ValueError(f"Expected {name} last dim {cols}, got {x.shape[1]}")


def _check_bias_gate(logit_bias: torch.Tensor | None, shared_gate_w: torch.Tensor | None,
                     E: int, H: int) -> None:
    """The kernels read E float32 biases and H bf16 shared-gate weights."""
    if logit_bias is not None and (logit_bias.dtype != torch.float32 or logit_bias.numel() != E):
        raise ValueError("logit_bias must be float32 [E]")
    if shared_gate_w is not None and (shared_gate_w.dtype != torch.bfloat16
                                      or shared_gate_w.numel() != H):
        raise ValueError("shared_gate_w must be bfloat16 with hidden elements")


def _check_blocks(sorted_ids: torch.Tensor, expert_ids: torch.Tensor, ntpp: torch.Tensor,
                  block_m: int) -> None:
    """align's outputs as the grouped GEMMs read them: expert_ids.numel() blocks of block_m
    sorted slot ids and the padded total."""
    for name, t in (("sorted_ids", sorted_ids), ("expert_ids", expert_ids), ("ntpp", ntpp)):
        if t.dtype != torch.int32:
            raise TypeError(f"{name} must be int32")
    if sorted_ids.numel() < expert_ids.numel() * block_m or ntpp.numel() < 1:
        raise ValueError(f"sorted_ids holds {sorted_ids.numel()} ids for {expert_ids.numel()} "
                         f"blocks of {block_m}")


# ----------------------------------------------------------------------------- dequant
def dequantize(qweight: torch.Tensor, qzeros: torch.Tensor, scales: torch.Tensor,
               g_idx: torch.Tensor | None = None, *, group_size: int = 128,
               linear_weight: bool = True, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """HIP dequant of one ([K/8, N]) or stacked ([E, K/8, N]) GPTQ projection.

    Bit-exact with dequantize_gptq_projection
    (src/mtp_expert_prefetch/repack/gptq_unpack.py:88-131)."""
    lib = _lib.load()
    squeeze = qweight.ndim == 2
    if squeeze:
        qweight, qzeros, scales = qweight[None], qzeros[None], scales[None]
        if g_idx is not None:
            g_idx = g_idx[None]
    _require_gpu(qweight, qzeros, scales, g_idx)
    if dtype not in OUT_DTYPES:
        raise ValueError(f"Unsupported dtype {dtype}")
    if qweight.ndim != 3 or qweight.dtype != torch.int32 or qzeros.dtype != torch.int32:
        raise TypeError("qweight [E, K/8, N] and qzeros must be int32")
    if scales.dtype != torch.float16:
        raise TypeError(f"scales must be float16, got {scales.dtype}")
    e, k8, n = qweight.shape
    k = k8 * 8
    if group_size <= 0 or k % group_size != 0:
        raise ValueError(f"group_size {group_size} does not divide in_features {k}")
    ng = k // group_size
    if tuple(scales.shape) != (e, ng, n) or tuple(qzeros.shape) != (e, ng, n // 8):
        raise ValueError(f"scales {tuple(scales.shape)} / qzeros {tuple(qzeros.shape)} do not "
                         f"match qweight {tuple(qweight.shape)} with group_size {group_size}")
    if g_idx is not None:
        if tuple(g_idx.shape) != (e, k):
            raise ValueError(f"g_idx {tuple(g_idx.shape)} must be [E, K] = {(e, k)}")
        lo, hi = (int(v) for v in torch.aminmax(g_idx))
        if lo < 0 or hi >= ng:  # the kernel reads the scales and zeros row g_idx[k]
            raise ValueError(f"g_idx out of range [{lo}, {hi}] for {ng} groups")
    out_shape = (e, n, k) if linear_weight else (e, k, n)
    out = torch.empty(out_shape, dtype=dtype, device=qweight.device)
    proj = _lib.GptqProj(qweight.data_ptr(), qzeros.data_ptr(), scales.data_ptr())
    gi = None
    if g_idx is not None:
        gi = g_idx.to(torch.int32).contiguous()
    _lib.check(lib.moe_dequant_v1(ctypes.byref(proj), _ptr(gi), e, k, n, group_size,
                                  1 if linear_weight else 0, OUT_DTYPES[dtype], out.data_ptr(),
                                  _stream()))
    return out[0] if squeeze else out


# ----------------------------------------------------------------------------- router
def router_topk(x: torch.Tensor, router_w: torch.Tensor, top_k: int = 8, *,
                logit_bias: torch.Tensor | None = None,
                shared_gate_w: torch.Tensor | None = None):
    """fp32 logits -> softmax -> top-k -> renormalise (bit-exact ids, ties to the lower id).

    Returns (topk_ids int32 [T, k], topk_weights fp32 [T, k], shared_gate fp32 [T] or None,
    logits fp32 [T, E])."""
    lib = _lib.load()
    _bf16_matrix(x, "input")
    _bf16_matrix(router_w, "router_w", x.shape[1])
    _require_gpu(x, router_w, logit_bias, shared_gate_w)
    T, E = x.shape[0], router_w.shape[0]
    if not 0 < top_k <= E:
        raise ValueError(f"top_k must be in [1, {E}], got {top_k}")
    dev = x.device
    logits = torch.empty(T, E + 1, dtype=torch.float32, device=dev)
    ids = torch.empty(T, top_k, dtype=torch.int32, device=dev)
    has_shared = shared_gate_w is not None
    w = torch.empty(T * top_k + (T if has_shared else 0), dtype=torch.float32, device=dev)
    if logit_bias is not None and (logit_bias.dtype != torch.float32 or logit_bias.numel() != E):
        raise ValueError("logit_bias must be float32 [E]")
    if has_shared:
        if shared_gate_w.dtype != torch.bfloat16 or shared_gate_w.numel() != x.shape[1]:
            raise ValueError("shared_gate_w must be bfloat16 with hidden elements")
    _lib.check(lib.moe_router_topk_v1(x.data_ptr(), T, x.shape[1], router_w.data_ptr(), E,
                                      _ptr(logit_bias), top_k, _ptr(shared_gate_w),
                                      logits.data_ptr(), ids.data_ptr(), w.data_ptr(), _stream()))
    topk_w = w[: T * top_k].view(T, top_k)
    shared = w[T * top_k:] if has_shared else None
    return ids, topk_w, shared, logits[:, :E]


# ----------------------------------------------------------------------------- align
def capacity_blocks(T: int, top_k: int, num_experts: int, has_shared: bool, block_m: int) -> int:
    return int(_lib.load().moe_capacity_blocks_v1(T, top_k, num_experts, int(has_shared), block_m))


def align(topk_ids: torch.Tensor, num_experts: int, block_m: int, *, has_shared: bool = False,
          capacity: int | None = None):
    """Block-padded expert-grouped slot permutation (vLLM moe_align_block_size format)."""
    lib = _lib.load()
    if topk_ids.dtype != torch.int32 or topk_ids.ndim != 2:
        raise TypeError("topk_ids must be int32 [T, k]")
    _require_gpu(topk_ids)
    T, k = topk_ids.shape
    cap = capacity if capacity is not None else capacity_blocks(T, k, num_experts, has_shared, block_m)
    dev = topk_ids.device
    sorted_ids = torch.empty(cap * block_m, dtype=torch.int32, device=dev)
    eids = torch.empty(cap, dtype=torch.int32, device=dev)
    ntpp = torch.empty(1, dtype=torch.int32, device=dev)
    _lib.check(lib.moe_align_v1(topk_ids.data_ptr(), T, k, num_experts, int(has_shared), block_m,
                                cap, sorted_ids.data_ptr(), eids.data_ptr(), ntpp.data_ptr(),
                                _stream()))
    return sorted_ids, eids, ntpp


# ----------------------------------------------------------------------------- GEMMs
def _block_m(path: int, T: int, top_k: int) -> int:
    if path == _lib.PATH_AUTO:
        path = _lib.PATH_PREFILL if T * top_k >= AUTO_PREFILL_SLOTS else _lib.PATH_DECODE
    return PREFILL_BLOCK_M if path == _lib.PATH_PREFILL else DECODE_BLOCK_M


def w1_gateup_silu(x, experts: MoeExperts, sorted_ids, expert_ids, ntpp, *, top_k: int,
                   shared: MoeExperts | None = None, path: str | int = "auto") -> torch.Tensor:
    lib = _lib.load()
    p = _path(path)
    _bf16_matrix(x, "input", experts.hidden_size)
    _require_gpu(x, sorted_ids, expert_ids, ntpp)
    _require_experts_on(x.device, experts, shared)
    T = x.shape[0]
    bm = _block_m(p, T, top_k)
    _check_blocks(sorted_ids, expert_ids, ntpp, bm)
    slots = T * top_k + (T if shared is not None else 0)
    h = torch.empty(slots, experts.intermediate_size, dtype=torch.bfloat16, device=x.device)
    ex = experts.struct()
    sh = shared.struct() if shared is not None else None
    _lib.check(lib.moe_w1_gateup_silu_v1(
        x.data_ptr(), T, top_k, ctypes.byref(ex), ctypes.byref(sh) if sh else None,
        sorted_ids.data_ptr(), expert_ids.data_ptr(), ntpp.data_ptr(), bm, expert_ids.numel(),
        h.data_ptr(), p, _stream()))
    return h


def w2_down(h, experts: MoeExperts, sorted_ids, expert_ids, ntpp, topk_weights_flat, *, T: int,
            top_k: int, shared: MoeExperts | None = None, path: str | int = "auto",
            ys: torch.Tensor | None = None) -> torch.Tensor:
    """Weighted W2 rows ys fp32 [slots, H]; rows of dropped slots are left as they were."""
    lib = _lib.load()
    p = _path(path)
    slots = T * top_k + (T if shared is not None else 0)
    _bf16_matrix(h, "h", experts.intermediate_size)
    if h.shape[0] < slots:
        raise ValueError(f"h has {h.shape[0]} rows for {slots} slots")
    if topk_weights_flat.dtype != torch.float32 or topk_weights_flat.numel() < slots:
        raise ValueError(f"topk_weights_flat must be float32 with at least {slots} elements")
    _require_gpu(h, sorted_ids, expert_ids, ntpp, topk_weights_flat)
    _require_experts_on(h.device, experts, shared)
    bm = _block_m(p, T, top_k)
    _check_blocks(sorted_ids, expert_ids, ntpp, bm)
    if ys is None:
        ys = torch.empty(h.shape[0], experts.hidden_size, dtype=torch.float32, device=h.device)
    elif (ys.dtype != torch.float32 or tuple(ys.shape) != (h.shape[0], experts.hidden_size)
          or not ys.is_contiguous()):
        raise ValueError("ys must be contiguous float32 [slots, hidden]")
    _require_gpu(h, ys)
    ex = experts.struct()
    sh = shared.struct() if shared is not None else None
    _lib.check(lib.moe_w2_down_v1(
        h.data_ptr(), T, top_k, ctypes.byref(ex), ctypes.byref(sh) if sh else None,
        sorted_ids.data_ptr(), expert_ids.data_ptr(), ntpp.data_ptr(), bm, expert_ids.numel(),
        topk_weights_flat.data_ptr(), ys.data_ptr(), p, _stream()))
    return ys


def moe_sum(ys: torch.Tensor, topk_ids: torch.Tensor, experts: MoeExperts,
            has_shared: bool = False) -> torch.Tensor:
    """Fixed-order fp32 sum of each token's weighted W2 rows -> bf16 [T, H]. Slots whose id is
    outside [0, E) or whose expert is not resident in a slot pool are skipped (w2_down leaves
    their rows unwritten)."""
    lib = _lib.load()
    if topk_ids.dtype != torch.int32 or topk_ids.ndim != 2:
        raise TypeError("topk_ids must be int32 [T, k]")
    _require_gpu(ys, topk_ids)
    T, top_k = topk_ids.shape
    H = ys.shape[1]
    if (ys.dtype != torch.float32 or ys.ndim != 2
            or ys.shape[0] < T * top_k + (T if has_shared else 0)):
        raise ValueError("ys must be float32 [T*k (+T), H]")
    out = torch.empty(T, H, dtype=torch.bfloat16, device=ys.device)
    _lib.check(lib.moe_sum_v1(ys.data_ptr(), T, top_k, H, int(has_shared), topk_ids.data_ptr(),
                              int(experts.num_experts), _ptr(experts.expert_row), out.data_ptr(),
                              _stream()))
    return out


# ----------------------------------------------------------------------------- decoder norm
def rmsnorm(res: torch.Tensor, weight: torch.Tensor, *, add: torch.Tensor | None = None,
            eps: float = 1e-6, out: torch.Tensor | None = None) -> torch.Tensor:
    """Residual add (in place into ``res`` when ``add`` is given) and the (1 + w) RMSNorm of
    mtp_rms_norm (src/mtp_expert_prefetch/mtp/extra_tensors.py:40-48) on the HIP kernel.

    res, add: bf16 [T, hidden]; weight bf16 [hidden]. Returns bf16 [T, hidden]."""
    lib = _lib.load()
    _bf16_matrix(res, "res")
    T, H = res.shape
    if add is not None:
        _bf16_matrix(add, "add", H)
        if add.shape[0] != T:
            raise ValueError(f"add has {add.shape[0]} rows for {T}")
    if weight.dtype != torch.bfloat16 or weight.numel() != H or not weight.is_contiguous():
        raise ValueError("weight must be a contiguous bfloat16 tensor of hidden elements")
    _require_gpu(res, add, weight)
    if out is None:
        out = torch.empty_like(res)
    elif out.shape != res.shape or out.dtype != torch.bfloat16 or not out.is_contiguous():
        raise ValueError("out must be a contiguous bf16 tensor shaped like res")
    _require_gpu(res, out)
    _lib.check(lib.moe_rmsnorm_v1(res.data_ptr(), _ptr(add), T, H, weight.data_ptr(), float(eps),
                                  out.data_ptr(), _stream()))
    return out


# ----------------------------------------------------------------------------- whole layer
def workspace_bytes(T: int, top_k: int, experts: MoeExperts, has_shared: bool,
                    path: str | int = "auto") -> int:
    ex = experts.struct()
    n = int(_lib.load().moe_layer_workspace_bytes_v1(T, top_k, ctypes.byref(ex), int(has_shared),
                                                     _path(path)))
    if n < 0:
        raise ValueError("invalid sizes for the workspace query")
    return n


def moe_layer(x: torch.Tensor, router_w: torch.Tensor, experts: MoeExperts, *, top_k: int = 8,
              logit_bias: torch.Tensor | None = None, shared: MoeExperts | None = None,
              shared_gate_w: torch.Tensor | None = None, path: str | int = "auto",
              workspace: torch.Tensor | None = None, return_routing: bool = False,
              out: torch.Tensor | None = None):
    """Routed MoE layer: router -> align -> W1 -> W2 -> sum (+ gated shared expert)."""
    lib = _lib.load()
    _bf16_matrix(x, "input", experts.hidden_size)
    _bf16_matrix(router_w, "router_w", experts.hidden_size)
    if router_w.shape[0] != experts.num_experts:
        raise ValueError(f"router_w has {router_w.shape[0]} rows for {experts.num_experts} experts")
    if (shared is None) != (shared_gate_w is None):
        raise ValueError("shared and shared_gate_w must be given together")
    _check_bias_gate(logit_bias, shared_gate_w, experts.num_experts, experts.hidden_size)
    _require_gpu(x, router_w, logit_bias, shared_gate_w)
    _require_experts_on(x.device, experts, shared)
    T = x.shape[0]
    p = _path(path)
    workspace = _workspace(workspace, workspace_bytes(T, top_k, experts, shared is not None, p),
                           x.device)
    if out is None:
        out = torch.empty_like(x)
    elif out.shape != x.shape or out.dtype != torch.bfloat16 or not out.is_contiguous():
        raise ValueError("out must be a contiguous bf16 tensor shaped like the input")
    _require_gpu(x, out)
    ids = torch.empty(T, top_k, dtype=torch.int32, device=x.device) if return_routing else None
    w = torch.empty(T, top_k, dtype=torch.float32, device=x.device) if return_routing else None
    ex = experts.struct()
    sh = shared.struct() if shared is not None else None
    _lib.check(lib.moe_layer_v1(
        x.data_ptr(), T, router_w.data_ptr(), _ptr(logit_bias), top_k, ctypes.byref(ex),
        ctypes.byref(sh) if sh else None, _ptr(shared_gate_w), workspace.data_ptr(),
        _nbytes(workspace), out.data_ptr(), _ptr(ids), _ptr(w), p, _stream()))
    if return_routing:
        return out, ids, w
    return out


def norm_layer(res: torch.Tensor, router_w: torch.Tensor, experts: MoeExperts,
               norm_w: torch.Tensor, *, add: torch.Tensor | None = None, eps: float = 1e-6,
               res_out: torch.Tensor | None = None, x_out: torch.Tensor | None = None,
               top_k: int = 8, logit_bias: torch.Tensor | None = None,
               shared: MoeExperts | None = None, shared_gate_w: torch.Tensor | None = None,
               path: str | int = "auto", workspace: torch.Tensor | None = None,
               out: torch.Tensor | None = None):
    """A decoder step: res_out = res + add, x = rmsnorm(res_out) * (1 + norm_w), then the routed
    layer on x (moe_norm_layer_v1; the bits of ``rmsnorm`` followed by ``moe_layer``). Returns
    (out, res_out, x). res_out defaults to a new tensor (a distinct buffer lets decode batches
    normalise inside the router); pass ``res`` itself to update it in place."""
    lib = _lib.load()
    _bf16_matrix(res, "res", experts.hidden_size)
    _bf16_matrix(router_w, "router_w", experts.hidden_size)
    T, H = res.shape
    if add is not None:
        _bf16_matrix(add, "add", H)
        if add.shape[0] != T:
            raise ValueError(f"add has {add.shape[0]} rows for {T}")
    if norm_w.dtype != torch.bfloat16 or norm_w.numel() != H or not norm_w.is_contiguous():
        raise ValueError("norm_w must be a contiguous bfloat16 tensor of hidden elements")
    if (shared is None) != (shared_gate_w is None):
        raise ValueError("shared and shared_gate_w must be given together")
    _check_bias_gate(logit_bias, shared_gate_w, experts.num_experts, experts.hidden_size)
    _require_gpu(res, add, norm_w, router_w, logit_bias, shared_gate_w)
    _require_experts_on(res.device, experts, shared)
    if res_out is None:
        res_out = torch.empty_like(res)
    if x_out is None:
        x_out = torch.empty_like(res)
    if out is None:
        out = torch.empty_like(res)
    for t, name in ((res_out, "res_out"), (x_out, "x_out"), (out, "out")):
        if t.shape != res.shape or t.dtype != torch.bfloat16 or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous bf16 tensor shaped like res")
    _require_gpu(res, res_out, x_out, out)
    p = _path(path)
    workspace = _workspace(workspace, workspace_bytes(T, top_k, experts, shared is not None, p),
                           res.device)
    ex = experts.struct()
    sh = shared.struct() if shared is not None else None
    _lib.check(lib.moe_norm_layer_v1(
        res.data_ptr(), _ptr(add), norm_w.data_ptr(), float(eps), res_out.data_ptr(),
        x_out.data_ptr(), T, router_w.data_ptr(), _ptr(logit_bias), top_k, ctypes.byref(ex),
        ctypes.byref(sh) if sh else None, _ptr(shared_gate_w), workspace.data_ptr(),
        _nbytes(workspace), out.data_ptr(), None, None, p, _stream()))
    return out, res_out, x_out


def fused_experts(x: torch.Tensor, topk_ids: torch.Tensor, topk_weights: torch.Tensor,
                  experts: MoeExperts, *, shared: MoeExperts | None = None,
                  shared_gate_w: torch.Tensor | None = None, path: str | int = "auto",
                  workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Experts with caller-given routing (ids int32 [T, k], weights fp32 [T, k])."""
    lib = _lib.load()
    _bf16_matrix(x, "input", experts.hidden_size)
    if topk_ids.dtype != torch.int32 or topk_weights.dtype != torch.float32:
        raise TypeError("topk_ids must be int32 and topk_weights float32")
    if topk_ids.shape != topk_weights.shape or topk_ids.ndim != 2 or topk_ids.shape[0] != x.shape[0]:
        raise ValueError("topk_ids/topk_weights must be [T, k] matching the input rows")
    if (shared is None) != (shared_gate_w is None):
        raise ValueError("shared and shared_gate_w must be given together")
    _check_bias_gate(None, shared_gate_w, experts.num_experts, experts.hidden_size)
    _require_gpu(x, topk_ids, topk_weights, shared_gate_w)
    _require_experts_on(x.device, experts, shared)
    T, k = topk_ids.shape
    p = _path(path)
    workspace = _workspace(workspace, workspace_bytes(T, k, experts, shared is not None, p),
                           x.device)
    out = torch.empty_like(x)
    ex = experts.struct()
    sh = shared.struct() if shared is not None else None
    _lib.check(lib.moe_fused_experts_v1(
        x.data_ptr(), T, topk_ids.data_ptr(), topk_weights.data_ptr(), k, ctypes.byref(ex),
        ctypes.byref(sh) if sh else None, _ptr(shared_gate_w), workspace.data_ptr(),
        _nbytes(workspace), out.data_ptr(), p, _stream()))
    return out


# ----------------------------------------------------------------------------- predictor
def predictor_workspace_bytes(T: int, num_heads: int, inner: int, num_experts: int, top_k: int) -> int:
    return int(_lib.load().moe_predictor_workspace_bytes_v1(T, num_heads, inner, num_experts, top_k))


def predictor_topk(h: torch.Tensor, w1: torch.Tensor, w2: torch.Tensor, top_k: int = 16, *,
                   workspace: torch.Tensor | None = None,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """Per-layer predicted experts: int32 [L, T, top_k] from h bf16 [T, H], w1 bf16 [L, D, H]
    (or [D, H] for one head), w2 bf16 [L, E, D] (or [E, D]).

    Each head computes bf16(silu(h . w1[l]^T)) . w2[l]^T in fp32 and keeps its top-k by
    (logit desc, id asc); the reference's per-layer predictor head
    (src/mtp_expert_prefetch/training/hidden_residual.py:44-106) simplified to hidden -> inner
    (SiLU) -> experts.
    """
    lib = _lib.load()
    if w1.dim() == 2:
        w1 = w1.unsqueeze(0)
    if w2.dim() == 2:
        w2 = w2.unsqueeze(0)
    _bf16_matrix(h, "hidden")
    if w1.dim() != 3 or w2.dim() != 3 or w1.shape[0] != w2.shape[0]:
        raise ValueError("w1 must be [L, D, H] and w2 [L, E, D] with the same L")
    L, D, H = w1.shape
    E = w2.shape[1]
    if H != h.shape[1] or w2.shape[2] != D:
        raise ValueError(f"predictor shapes: h {tuple(h.shape)}, w1 {tuple(w1.shape)}, w2 {tuple(w2.shape)}")
    for t, name in ((w1, "w1"), (w2, "w2")):
        if t.dtype != torch.bfloat16 or not t.is_contiguous():
            raise TypeError(f"{name} must be contiguous bf16")
    _require_gpu(h, w1, w2)
    T = h.shape[0]
    # a negative size (invalid sizes) leaves the error to the entry point's own checks
    workspace = _workspace(workspace, predictor_workspace_bytes(T, L, D, E, top_k), h.device)
    if out is None:
        out = torch.empty(L, T, top_k, dtype=torch.int32, device=h.device)
    elif out.dtype != torch.int32 or out.shape != (L, T, top_k) or not out.is_contiguous():
        raise ValueError("out must be contiguous int32 [L, T, top_k]")
    _require_gpu(h, out)
    _lib.check(lib.moe_predictor_v1(h.data_ptr(), T, H, L, w1.data_ptr(), D, w2.data_ptr(), E,
                                    top_k, workspace.data_ptr(), _nbytes(workspace),
                                    out.data_ptr(), _stream()))
    return out


# ----------------------------------------------------------------------------- by expert and back
def _call(entry: str, device: torch.device, *args) -> None:
    """An entry point on ``device`` (which need not be the current one) and its current stream.
    The raw queries take 0.1 us; torch.cuda.current_stream builds an object in 3 us, a quarter of a
    small call's time on the host, and torch.cuda.current_device takes 3 us on autograd's thread."""
    fn = getattr(_lib.load(), entry)
    index = device.index
    if index == torch._C._cuda_getDevice():
        code = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(device):
            code = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if code:
        _lib.check(code)


def _rows_2d(x: torch.Tensor, name: str) -> int:
    """The dtype code of a [rows, columns] tensor of a supported type."""
    code = OUT_DTYPES.get(x.dtype)
    if code is None:
        raise TypeError(f"{name} must be bfloat16, float16 or float32, got {x.dtype}")
    shape = x.shape
    if len(shape) != 2 or shape[0] >> 31 or shape[1] >> 31:  # sizes are int32 in the library
        raise ValueError(f"{name} must be 2D with sizes below 2^31, got {tuple(shape)}")
    return code


# The calls below go through their autograd function where a gradient may be asked for, and inside a dual
# level, where the function refuses a dual tensor (past it the tangent would be lost). Each looks at
# its own inputs: with a helper for all of them an int8_linear of one row took 9.1 us instead of 8.8.


def _refuse_dual(*grads: torch.Tensor | None) -> None:
    """A backward pass carries no forward-mode derivative of its incoming gradients either."""
    if forward_ad._current_level >= 0:
        for g in grads:
            if g is not None and forward_ad.unpack_dual(g).tangent is not None:
                raise NotImplementedError("the backward pass has no jvp: dual gradients are refused")


class Dispatch(NamedTuple):
    """Token rows sorted by expert (``dispatch_tokens``)."""

    rows: torch.Tensor      # [T * k, H]: expert by expert, slots in order; dropped slots' zeros last
    offsets: torch.Tensor   # int32 [E + 1]: first row of each expert; offsets[E] rows are in use
    row_slot: torch.Tensor  # int32 [T * k]: slot t * k + i of each row
    slot_row: torch.Tensor  # int32 [T, k]: row of each slot; ~row (negative) where it is dropped


def _dispatch(x, topk_ids, num_experts):
    T, H = x.shape
    k = topk_ids.shape[1]
    dev = x.device
    rows = torch.empty(T * k, H, dtype=x.dtype, device=dev)
    offsets = torch.empty(num_experts + 1, dtype=torch.int32, device=dev)
    row_slot = torch.empty(T * k, dtype=torch.int32, device=dev)
    slot_row = torch.empty_like(topk_ids)
    need = _lib.load().moe_dispatch_workspace_bytes_v1(T, k, num_experts)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need > 0 else None
    _call("moe_dispatch_v1", dev, x.data_ptr(), T, H, OUT_DTYPES[x.dtype], topk_ids.data_ptr(), k,
          num_experts, _ptr(ws), need, rows.data_ptr(), offsets.data_ptr(),
          row_slot.data_ptr(), slot_row.data_ptr())
    return rows, offsets, row_slot, slot_row


def _combine(rows, slot_row, topk_weights):
    T, k = slot_row.shape
    out = torch.empty(T, rows.shape[1], dtype=rows.dtype, device=rows.device)
    _call("moe_combine_v1", rows.device, rows.data_ptr(), T, k, rows.shape[1],
          OUT_DTYPES[rows.dtype], slot_row.data_ptr(), _ptr(topk_weights), out.data_ptr())
    return out


class _DispatchFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, topk_ids, num_experts):
        rows, offsets, row_slot, slot_row = _dispatch(x, topk_ids, num_experts)
        ctx.mark_non_differentiable(offsets, row_slot, slot_row)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(slot_row)
        return rows, offsets, row_slot, slot_row

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_rows, *_):
        if grad_rows is None:
            return None, None, None
        _refuse_dual(grad_rows)
        return _combine(grad_rows.contiguous(), ctx.saved_tensors[0], None), None, None


class _CombineFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, slot_row, topk_weights):
        ctx.save_for_backward(rows, slot_row, topk_weights)
        return _combine(rows, slot_row, topk_weights)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        rows, slot_row, topk_weights = ctx.saved_tensors
        _refuse_dual(grad_out)
        want_rows, _, want_weights = ctx.needs_input_grad
        grad_out = grad_out.contiguous()
        T, k = slot_row.shape
        drows = torch.empty_like(rows) if want_rows else None
        dweights = torch.empty_like(topk_weights) if want_weights else None
        _call("moe_combine_backward_v1", rows.device, grad_out.data_ptr(), rows.data_ptr(), T, k,
              rows.shape[1], OUT_DTYPES[rows.dtype], slot_row.data_ptr(), topk_weights.data_ptr(),
              _ptr(drows), _ptr(dweights))
        return drows, None, dweights


def dispatch_tokens(x: torch.Tensor, topk_ids: torch.Tensor, num_experts: int) -> Dispatch:
    """Token rows sorted by expert, for products of the caller's own over each expert's rows.

    x [T, H] (bf16, fp16 or fp32), topk_ids int32 [T, k]. Rows are ordered by (expert, slot), a
    stable sort; a slot whose id is outside [0, num_experts) is dropped and takes a row of zeros
    behind offsets[num_experts]. Differentiable in x: its gradient sums the rows' over each token's
    kept slots in fp32. An expert may occur twice in a token's ids: each slot has its own row."""
    _rows_2d(x, "x")
    if topk_ids.dtype != torch.int32 or topk_ids.ndim != 2:
        raise TypeError("topk_ids must be int32 [T, k]")
    if topk_ids.shape[0] != x.shape[0] or topk_ids.shape[1] > 64:
        raise ValueError(f"topk_ids must be [{x.shape[0]}, k] with k <= 64, got "
                         f"{tuple(topk_ids.shape)}")
    if not 1 <= num_experts <= 512:
        raise ValueError(f"num_experts must lie in [1, 512], got {num_experts}")
    _require_gpu(x, topk_ids)
    if (x.requires_grad and torch.is_grad_enabled()) or forward_ad._current_level >= 0:
        return Dispatch(*_DispatchFn.apply(x, topk_ids, int(num_experts)))
    return Dispatch(*_dispatch(x, topk_ids, int(num_experts)))


def combine_tokens(rows: torch.Tensor, slot_row: torch.Tensor,
                   topk_weights: torch.Tensor) -> torch.Tensor:
    """The experts' rows back at their tokens: out[t] = sum_i topk_weights[t, i] *
    rows[slot_row[t, i]] over the kept slots, in slot order in fp32, rounded once to rows' type.

    rows [T * k, H] and slot_row int32 [T, k] as ``dispatch_tokens`` gives them (every row belongs
    to one slot; a slot is dropped by giving ``dispatch_tokens`` an id outside the experts, not by
    changing slot_row), topk_weights fp32 [T, k]. What a dropped slot's row and weight hold is not
    looked at. Differentiable in rows (dropped slots' rows: zeros) and in topk_weights."""
    _rows_2d(rows, "rows")
    if slot_row.dtype != torch.int32 or topk_weights.dtype != torch.float32:
        raise TypeError("slot_row must be int32 and topk_weights float32")
    if slot_row.ndim != 2 or slot_row.shape != topk_weights.shape:
        raise ValueError("slot_row and topk_weights must be [T, k]")
    if rows.shape[0] != slot_row.numel():
        raise ValueError(f"rows has {rows.shape[0]} rows for {slot_row.numel()} slots")
    _require_gpu(rows, slot_row, topk_weights)
    if (((rows.requires_grad or topk_weights.requires_grad) and torch.is_grad_enabled())
            or forward_ad._current_level >= 0):
        return _CombineFn.apply(rows, slot_row, topk_weights)
    return _combine(rows, slot_row, topk_weights)


# ----------------------------------------------------------------------------- int8 products
class _NoGradientFn(torch.autograd.Function):
    """The result of a call without a derivative, one of whose inputs is part of a graph: a backward pass
    that reaches the call raises. Detached from them it would lose their gradients in silence."""

    @staticmethod
    def forward(ctx, out, name, *inputs):
        ctx.name = name
        ctx.mark_dirty(out)
        return out

    @staticmethod
    def backward(ctx, *_):
        raise NotImplementedError(f"{ctx.name} has no gradient: detach its inputs where it is to end "
                                  "there")


def quantize_tokens(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """int8 rows and their scales: scale = max|x[t]| / 127, q = x / scale rounded half to even.

    x [T, K] bf16, fp16 or fp32 -> (int8 [T, K], fp32 [T]). A row that holds an infinity or NaN
    gets q = 0 and a scale that is not finite, so its products are NaN. No gradient: a backward pass
    through the scale raises (q is an integer, of which there is none)."""
    code = _rows_2d(x, "x")
    _require_gpu(x)
    T, K = x.shape
    q = torch.empty(T, K, dtype=torch.int8, device=x.device)
    scale = torch.empty(T, dtype=torch.float32, device=x.device)
    _call("moe_quantize_tokens_v1", x.device, x.data_ptr(), T, K, code, q.data_ptr(),
          scale.data_ptr())
    if (x.requires_grad and torch.is_grad_enabled()) or forward_ad._current_level >= 0:
        scale = _NoGradientFn.apply(scale, "quantize_tokens", x)
    return q, scale


def _check_int8(weight, weight_scale, bias, K: int, dtype: torch.dtype) -> None:
    if weight.dtype != torch.int8 or weight_scale.dtype != torch.float32:
        raise TypeError(f"weight must be int8 and weight_scale float32, got {weight.dtype} and "
                        f"{weight_scale.dtype}")
    if weight.ndim != 2 or weight.shape[1] != K or tuple(weight_scale.shape) != weight.shape[:1]:
        raise ValueError(f"weight must be [N, {K}] and weight_scale [N], got "
                         f"{tuple(weight.shape)} and {tuple(weight_scale.shape)}")
    if max(weight.shape) >= 1 << 31:
        raise ValueError(f"weight's sizes must be below 2^31, got {tuple(weight.shape)}")
    if bias is not None and (bias.dtype != dtype or tuple(bias.shape) != weight.shape[:1]):
        raise ValueError(f"bias must be {dtype} [N]")


def int8_matmul(q: torch.Tensor, q_scale: torch.Tensor, weight: torch.Tensor,
                weight_scale: torch.Tensor, *, bias: torch.Tensor | None = None,
                dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """Product of int8 rows and int8 weights with a scale for each token and each channel:
    out[t, n] = (sum_k q[t, k] * weight[n, k]) * q_scale[t] * weight_scale[n] (+ bias[n]), the sum
    exact in 32 bits, the rest fp32, rounded once to ``dtype``.

    q int8 [T, K], q_scale fp32 [T], weight int8 [N, K], weight_scale fp32 [N], bias [N] of
    ``dtype``. K is a multiple of 16, at most 65536. No gradient: a backward pass that reaches the
    call raises."""
    if dtype not in OUT_DTYPES:
        raise TypeError(f"dtype must be bfloat16, float16 or float32, got {dtype}")
    if q.dtype != torch.int8 or q_scale.dtype != torch.float32:
        raise TypeError("q must be int8 and q_scale float32")
    if q.ndim != 2 or tuple(q_scale.shape) != q.shape[:1] or q.shape[0] >= 1 << 31:
        raise ValueError("q must be [T, K] with T below 2^31 and q_scale [T]")
    T, K = q.shape
    _check_int8(weight, weight_scale, bias, K, dtype)
    _require_gpu(q, q_scale, weight, weight_scale, bias)
    N = weight.shape[0]
    out = torch.empty(T, N, dtype=dtype, device=q.device)
    _call("moe_int8_matmul_v1", q.device, q.data_ptr(), q_scale.data_ptr(), T, K,
          weight.data_ptr(), weight_scale.data_ptr(), N, _ptr(bias), OUT_DTYPES[dtype],
          out.data_ptr())
    if ((q_scale.requires_grad or weight_scale.requires_grad or (bias is not None and bias.requires_grad))
            and torch.is_grad_enabled()) or forward_ad._current_level >= 0:
        out = _NoGradientFn.apply(out, "int8_matmul", q_scale, weight_scale, bias)
    return out


def int8_linear(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, *,
                bias: torch.Tensor | None = None) -> torch.Tensor:
    """A linear layer on int8 products: the values of ``quantize_tokens(x)`` followed by
    ``int8_matmul``, in x's type. x [T, K], weight int8 [N, K], weight_scale fp32 [N]. No gradient: a
    backward pass that reaches the call raises."""
    code = _rows_2d(x, "x")
    T, K = x.shape
    _check_int8(weight, weight_scale, bias, K, x.dtype)
    _require_gpu(x, weight, weight_scale, bias)
    N = weight.shape[0]
    dev = x.device
    need = _lib.load().moe_int8_linear_workspace_bytes_v1(T, K)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need > 0 else None
    out = torch.empty(T, N, dtype=x.dtype, device=dev)
    _call("moe_int8_linear_v1", dev, x.data_ptr(), T, K, code, weight.data_ptr(),
          weight_scale.data_ptr(), N, _ptr(bias), _ptr(ws), need, out.data_ptr())
    if ((x.requires_grad or weight_scale.requires_grad or (bias is not None and bias.requires_grad))
            and torch.is_grad_enabled()) or forward_ad._current_level >= 0:
        out = _NoGradientFn.apply(out, "int8_linear", x, weight_scale, bias)
    return out


def int8_experts_workspace_bytes(T: int, top_k: int, experts: Int8Experts,
                                 dtype: torch.dtype = torch.bfloat16) -> int:
    if T >> 31 or top_k >> 31:  # sizes are int32 in the library
        raise ValueError(f"T and top_k must lie in [0, 2^31), got {T} and {top_k}")
    ex = experts.struct()
    n = int(_lib.load().moe_int8_experts_workspace_bytes_v1(T, top_k, ctypes.byref(ex),
                                                            OUT_DTYPES[dtype]))
    if n < 0:
        raise ValueError(_lib.load().moe_w4a16_last_error().decode("utf-8", "replace"))
    return n


def int8_experts(x: torch.Tensor, topk_ids: torch.Tensor, topk_weights: torch.Tensor,
                 experts: Int8Experts, *, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Routed int8 experts with caller-given routing: the int8 counterpart of ``fused_experts``.

    Every kept slot's token is quantised and multiplied by the expert's gate and up projections,
    h = silu(g) * u is rounded to x's type, quantised and multiplied by down; the slots' rows come
    back as in ``combine_tokens``. x [T, H] bf16, fp16 or fp32; topk_ids int32 and topk_weights
    fp32 [T, k]; a slot whose id is outside [0, E) contributes nothing. A shared expert goes in as
    one more expert of the stacks, with its id and gate as one more slot of every token. No gradient:
    a backward pass that reaches the call raises."""
    code = _rows_2d(x, "x")
    if x.shape[1] != experts.hidden_size:
        raise ValueError(f"Expected x last dim {experts.hidden_size}, got {x.shape[1]}")
    if topk_ids.dtype != torch.int32 or topk_weights.dtype != torch.float32:
        raise TypeError("topk_ids must be int32 and topk_weights float32")
    if topk_ids.shape != topk_weights.shape or topk_ids.ndim != 2 or topk_ids.shape[0] != x.shape[0]:
        raise ValueError("topk_ids/topk_weights must be [T, k] matching the input rows")
    _require_gpu(x, topk_ids, topk_weights)
    if experts.device != x.device:
        raise ValueError(f"expert weights on {experts.device}, activations on {x.device}")
    T, k = topk_ids.shape
    ex = experts.struct()
    need = int(_lib.load().moe_int8_experts_workspace_bytes_v1(T, k, ctypes.byref(ex), code))
    # a negative size (invalid sizes) leaves the error to the entry point's own checks
    workspace = _workspace(workspace, need, x.device)
    out = torch.empty_like(x)
    _call("moe_int8_experts_v1", x.device, x.data_ptr(), T, code, topk_ids.data_ptr(),
          topk_weights.data_ptr(), k, ctypes.byref(ex), workspace.data_ptr(), _nbytes(workspace),
          out.data_ptr())
    scales = experts.gate_scale, experts.up_scale, experts.down_scale
    if ((x.requires_grad or topk_weights.requires_grad or any(s.requires_grad for s in scales))
            and torch.is_grad_enabled()) or forward_ad._current_level >= 0:
        out = _NoGradientFn.apply(out, "int8_experts", x, topk_weights, *scales)
    return out


# ----------------------------------------------------------------------------- norms around a block
GATE_NONE, GATE_TOKEN, GATE_CHANNEL, GATE_FULL = range(4)


def _block_norm(y, res, post_w, gate, pre_w, kind, res_scale, branch_scale, eps):
    T, H = y.shape
    res_out = torch.empty_like(res)
    x_out = torch.empty_like(res) if pre_w is not None else None
    _call("moe_block_norm_v1", y.device, y.data_ptr(), res.data_ptr(), T, H, OUT_DTYPES[y.dtype],
          _ptr(post_w), _ptr(gate), kind, res_scale, branch_scale, _ptr(pre_w), eps,
          res_out.data_ptr(), _ptr(x_out))
    return res_out, x_out


class _BlockNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, res, post_w, gate, pre_w, kind, res_scale, branch_scale, eps):
        res_out, x_out = _block_norm(y, res, post_w, gate, pre_w, kind, res_scale, branch_scale, eps)
        ctx.save_for_backward(y, res_out, post_w, gate, pre_w)
        ctx.consts = (kind, res_scale, branch_scale, eps)
        ctx.set_materialize_grads(False)
        return res_out if x_out is None else (res_out, x_out)

    @staticmethod
    @once_differentiable
    def backward(ctx, dres_out, dx=None):
        y, res_out, post_w, gate, pre_w = ctx.saved_tensors
        kind, res_scale, branch_scale, eps = ctx.consts
        if dres_out is None and dx is None:
            return (None,) * 9
        _refuse_dual(dres_out, dx)
        T, H = y.shape
        make = torch.empty_like if T > 0 else torch.zeros_like
        want_y, want_res, want_post, want_gate, want_pre = ctx.needs_input_grad[:5]
        dy = make(y) if want_y else None
        dres = make(res_out) if want_res else None
        dpost = make(post_w) if want_post else None
        dgate = make(gate) if want_gate else None
        dpre = make(pre_w) if want_pre else None
        if T > 0:
            if dres_out is not None:
                dres_out = dres_out.contiguous()
            if dx is not None:
                dx = dx.contiguous()
            elif want_pre:
                dpre.zero_()
            ws, need = None, 0
            if want_post or want_pre or kind == GATE_CHANNEL:
                need = _lib.load().moe_block_norm_workspace_bytes_v1(T, H)
                ws = torch.empty(need, dtype=torch.uint8, device=y.device)
            _call("moe_block_norm_backward_v1", y.device, y.data_ptr(), res_out.data_ptr(), T, H,
                  OUT_DTYPES[y.dtype], _ptr(post_w), _ptr(gate), kind, res_scale, branch_scale,
                  _ptr(pre_w), eps, _ptr(dres_out), _ptr(dx), _ptr(ws), need, _ptr(dy), _ptr(dres),
                  _ptr(dpost), _ptr(dgate), _ptr(dpre) if dx is not None else None)
        return dy, dres, dpost, dgate, dpre, None, None, None, None


def block_norm(y: torch.Tensor, res: torch.Tensor, *, post_w: torch.Tensor | None = None,
               gate: torch.Tensor | None = None, res_scale: float = 1.0,
               branch_scale: float = 1.0, pre_w: torch.Tensor | None = None,
               eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor | None]:
    """The norm behind a block, its gate, the scaled residual and the next block's norm at once:

        p = y * rsqrt(mean(y^2) + eps) * (1 + post_w)        (p = y without post_w)
        res_out = res_scale * res + branch_scale * gate * p
        x = res_out * rsqrt(mean(res_out^2) + eps) * (1 + pre_w)   (None without pre_w)

    with the (1 + w) scaling of ``rmsnorm``. y (the block's output) and res (the residual stream)
    [T, H], post_w and pre_w [H], gate [H] (per channel), [T, 1] (per token) or [T, H], all of one
    type (bf16, fp16 or fp32); H up to 8192. res_out is rounded to the type before x is computed
    from it. Returns (res_out, x); differentiable in y, res, post_w, gate and pre_w."""
    _rows_2d(y, "y")
    T, H = y.shape
    if res.shape != y.shape or res.dtype != y.dtype:
        raise ValueError(f"res must be {y.dtype} {tuple(y.shape)}, got {res.dtype} "
                         f"{tuple(res.shape)}")
    for name, w in (("post_w", post_w), ("pre_w", pre_w)):
        if w is not None and (w.dtype != y.dtype or tuple(w.shape) != (H,)):
            raise ValueError(f"{name} must be {y.dtype} [{H}], got {w.dtype} {tuple(w.shape)}")
    kind = GATE_NONE
    if gate is not None:
        kinds = {(T, 1): GATE_TOKEN, (H,): GATE_CHANNEL, (T, H): GATE_FULL}
        kind = kinds.get(tuple(gate.shape), GATE_NONE)
        if kind == GATE_NONE or gate.dtype != y.dtype:
            raise ValueError(f"gate must be {y.dtype} [{H}], [{T}, 1] or [{T}, {H}], got "
                             f"{gate.dtype} {tuple(gate.shape)}")
    _require_gpu(y, res, post_w, gate, pre_w)
    scales = (kind, float(res_scale), float(branch_scale), float(eps))
    if ((y.requires_grad or res.requires_grad or (post_w is not None and post_w.requires_grad)
         or (gate is not None and gate.requires_grad) or (pre_w is not None and pre_w.requires_grad))
            and torch.is_grad_enabled()) or forward_ad._current_level >= 0:
        out = _BlockNormFn.apply(y, res, post_w, gate, pre_w, *scales)
        return out if pre_w is not None else (out, None)
    return _block_norm(y, res, post_w, gate, pre_w, *scales)
