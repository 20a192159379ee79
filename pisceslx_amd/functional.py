"""Functional entry points over libyvmoe: torch allocates, the HIP library computes.

Every function runs on the tensors' CUDA (HIP) device and on torch's current stream; none
of them has a CPU or PyTorch fallback — a call on CPU tensors raises.
"""
from __future__ import annotations

import ctypes
import functools
import threading
import weakref
from dataclasses import dataclass
from typing import Optional

import torch
from torch.autograd import forward_ad

from . import _lib
from .quant import Fp8Rows, PackedExperts, PackedFp8Linear, PackedLinear


def _act(dtype: torch.dtype) -> int:
    if dtype == torch.bfloat16:
        return _lib.ACT_BF16
    if dtype == torch.float32:
        return _lib.ACT_F32
    raise ValueError(f"activation dtype {dtype} is not supported (bfloat16 or float32)")


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _stream(device: torch.device):
    """The handle of torch's current stream on a tensor's device (without the Stream object that
    torch.cuda.current_stream builds: 0.1 us instead of 1.9 on every call)."""
    return torch._C._cuda_getCurrentRawStream(device.index)


def _require_cuda(*ts: Optional[torch.Tensor]) -> torch.device:
    dev = None
    for t in ts:
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError("libyvmoe computes on the GPU only: got a CPU tensor")
        if not t.is_contiguous():
            raise ValueError("libyvmoe needs contiguous tensors")
        dev = t.device
    return dev


def router_ld(num_experts: int, act: int) -> int:
    ep = (num_experts + 15) // 16 * 16
    return ep + (3 if act == _lib.ACT_BF16 else 1) * _lib.PREDICTOR_DIM


@dataclass
class RouterState:
    """Device tensors of one YvStableMoEGate, packed for the router GEMM."""

    num_experts: int
    hidden: int
    top_k: int
    fixed_shape_mode: bool
    dynamic_capacity: bool
    min_capacity: int
    capacity_factor: float
    w_router: torch.Tensor
    b1: Optional[torch.Tensor]
    w2: Optional[torch.Tensor]
    b2: Optional[torch.Tensor]
    bias: Optional[torch.Tensor]

    def struct(self) -> _lib.Router:
        return _lib.Router(self.num_experts, self.hidden, self.top_k, int(self.fixed_shape_mode),
                           int(self.dynamic_capacity), self.min_capacity, float(self.capacity_factor),
                           _ptr(self.w_router), _ptr(self.b1), _ptr(self.w2), _ptr(self.b2),
                           _ptr(self.bias))


@dataclass
class Routing:
    weights: torch.Tensor   # [N, k] fp32
    indices: torch.Tensor   # [N, k] int64
    counts: torch.Tensor    # [E] int32
    offsets: torch.Tensor   # [E+1] int32
    perm: torch.Tensor      # [N*k] int32
    pos: torch.Tensor       # [N*k] int32
    capacity: torch.Tensor  # [1] int32

    @staticmethod
    def empty(N: int, E: int, k: int, device) -> "Routing":
        i32 = dict(dtype=torch.int32, device=device)
        return Routing(torch.empty(N, k, dtype=torch.float32, device=device),
                       torch.empty(N, k, dtype=torch.int64, device=device),
                       torch.empty(E, **i32), torch.empty(E + 1, **i32),
                       torch.empty(N * k, **i32), torch.empty(N * k, **i32),
                       torch.empty(1, **i32))

    @staticmethod
    def lazy(N: int, E: int, k: int, device) -> "Routing":
        """:meth:`empty` with the five int32 tensors in one allocation, made when they are read."""
        return _LazyRouting(N, E, k, device)

    def struct(self) -> _lib.Routing:
        return _lib.Routing(self.weights.data_ptr(), self.indices.data_ptr(), self.counts.data_ptr(),
                            self.offsets.data_ptr(), self.perm.data_ptr(), self.pos.data_ptr(),
                            self.capacity.data_ptr())


class _LazyRouting(Routing):
    _PARTS = ("counts", "offsets", "perm", "pos", "capacity")

    def __init__(self, N: int, E: int, k: int, device):
        self.weights = torch.empty(N, k, dtype=torch.float32, device=device)
        self.indices = torch.empty(N, k, dtype=torch.int64, device=device)
        self._lengths = (E, E + 1, N * k, N * k, 1)
        at, self._starts = 0, []
        for n in self._lengths:
            self._starts.append(at)
            at += (n + 63) // 64 * 64
        self._rest = torch.empty(at, dtype=torch.int32, device=device)

    def __getattr__(self, name):  # called for what is not set yet
        if name not in self._PARTS:
            raise AttributeError(name)
        i = self._PARTS.index(name)
        t = self._rest[self._starts[i]:self._starts[i] + self._lengths[i]]
        setattr(self, name, t)
        return t

    def struct(self) -> _lib.Routing:
        p = self._rest.data_ptr()
        return _lib.Routing(self.weights.data_ptr(), self.indices.data_ptr(), *(p + 4 * s for s in self._starts))


def workspace_bytes(n_tokens: int, act: int, router: RouterState,
                    experts: Optional[PackedExperts] = None) -> int:
    r = router.struct()
    e = experts.struct() if experts is not None else None
    return int(_lib.lib().yvmoe_workspace_bytes(n_tokens, act, ctypes.byref(r),
                                                ctypes.byref(e) if e is not None else None))


def _workspace(nbytes: int, device) -> torch.Tensor:
    return torch.empty(max(nbytes, 256), dtype=torch.uint8, device=device)


def router_logits(x2d: torch.Tensor, router: RouterState) -> torch.Tensor:
    """[N, ld] fp32: gate logits in columns [0, E), predictor first-layer terms after Ep."""
    dev = _require_cuda(x2d, router.w_router)
    act = _act(x2d.dtype)
    N = x2d.shape[0]
    ld = router_ld(router.num_experts, act)
    out = torch.empty(N, ld, dtype=torch.float32, device=dev)
    r = router.struct()
    ws = _workspace(int(_lib.lib().yvmoe_router_workspace_bytes(N, act, ctypes.byref(r))), dev)
    _lib.check(_lib.lib().yvmoe_router_logits(x2d.data_ptr(), act, N, ctypes.byref(r),
                                               out.data_ptr(), ld, ws.data_ptr(), ws.numel(),
                                               _stream(dev)),
               "yvmoe_router_logits")
    return out


def route(logits: torch.Tensor, router: RouterState, predictor: bool = True,
          capacity_override: int = -1) -> Routing:
    """Routing from fp32 logits [N, ld] (first E columns are the gate logits).

    ``predictor`` says the predictor columns follow at column Ep (as router_logits returns);
    pass False for plain [N, E] logits together with a capacity override or a fixed-mode gate.
    """
    dev = _require_cuda(logits)
    if logits.dtype != torch.float32:
        raise ValueError("routing needs fp32 logits")
    N, ld = logits.shape
    E, k = router.num_experts, router.top_k
    out = Routing.empty(N, E, k, dev)
    ws = _workspace(workspace_bytes(N, _lib.ACT_F32, router), dev)
    r = router.struct()
    o = out.struct()
    Ep = (E + 15) // 16 * 16
    pred_ptr = logits.data_ptr() + Ep * 4 if (predictor and N > 0) else None
    _lib.check(_lib.lib().yvmoe_route(logits.data_ptr() if N > 0 else None, ld, pred_ptr, N,
                                       ctypes.byref(r), capacity_override, ctypes.byref(o),
                                       ws.data_ptr(), ws.numel(), _stream(dev)), "yvmoe_route")
    return out


def expert_ffn(x2d: torch.Tensor, experts: PackedExperts, routing: Routing, top_k: int,
               workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y [N*k + S*N, H]: expert outputs in expert-sorted order, then the shared experts.

    Reads the routing's offsets and permutation only; ``workspace`` is scratch (allocated
    here when None or too small)."""
    dev = _require_cuda(x2d, *experts.tensors())
    act = _act(x2d.dtype)
    N = x2d.shape[0]
    R = N * top_k + experts.num_shared * N
    y = torch.empty(R, experts.hidden, dtype=x2d.dtype, device=dev)
    e = experts.struct()
    o = routing.struct()
    r = _lib.Router(experts.num_routed, experts.hidden, top_k, 0, 0, 0, 1.0, None, None, None,
                    None, None)
    need = int(_lib.lib().yvmoe_workspace_bytes(N, act, ctypes.byref(r), ctypes.byref(e)))
    if workspace is None or workspace.numel() < need:
        workspace = _workspace(need, dev)
    _lib.check(_lib.lib().yvmoe_expert_ffn(x2d.data_ptr(), act, N, top_k, ctypes.byref(e),
                                            ctypes.byref(o), y.data_ptr(), workspace.data_ptr(),
                                            workspace.numel(), _stream(dev)), "yvmoe_expert_ffn")
    return y


def dispatch_workspace_bytes(n_tokens: int, act: int, slots: int, experts: PackedExperts) -> int:
    e = experts.struct()
    return int(_lib.lib().yvmoe_dispatch_workspace_bytes(n_tokens, act, slots, ctypes.byref(e)))


def dispatch(x2d: torch.Tensor, routing_weights: torch.Tensor, expert_indices: torch.Tensor,
             experts: PackedExperts, want_expert_outputs: bool = False,
             workspace: Optional[torch.Tensor] = None):
    """Dispatch of an external routing (yvmoe_dispatch): grouped SwiGLU of the routed experts
    over every (token, slot) of ``expert_indices`` [N, k] int64 with ``routing_weights``
    [N, k] (fp32 or bf16), combined per token. Nothing synchronizes with the host.

    Returns (out [N, H], counts [E] int32, offsets [E+1] int32, invalid [1] int32 = number of
    slots whose index lies outside [0, E), expert outputs [N*k, H] in expert-sorted order or
    None).
    """
    dev = _require_cuda(x2d, routing_weights, expert_indices, *experts.tensors())
    act = _act(x2d.dtype)
    N, H = x2d.shape
    if H != experts.hidden:
        raise ValueError(f"hidden size {H} does not match the experts ({experts.hidden})")
    if expert_indices.dtype != torch.int64 or expert_indices.dim() != 2 or expert_indices.shape[0] != N:
        raise ValueError("expert_indices must be int64 [N, k]")
    k = expert_indices.shape[1]
    if tuple(routing_weights.shape) != (N, k):
        raise ValueError(f"routing_weights must be [N, k] = [{N}, {k}]")
    wdt = _act(routing_weights.dtype)
    E = experts.num_routed
    out = torch.empty_like(x2d)
    counts = torch.empty(E, dtype=torch.int32, device=dev)
    offsets = torch.empty(E + 1, dtype=torch.int32, device=dev)
    invalid = torch.empty(1, dtype=torch.int32, device=dev)
    y = torch.empty(N * k, H, dtype=x2d.dtype, device=dev) if want_expert_outputs else None
    need = dispatch_workspace_bytes(N, act, k, experts)
    if need == 0:
        raise ValueError(f"yvmoe_dispatch_workspace_bytes rejected k={k}")
    if workspace is None or workspace.numel() < need:
        workspace = _workspace(need, dev)
    e = experts.struct()
    _lib.check(_lib.lib().yvmoe_dispatch(
        x2d.data_ptr() if N > 0 else None, act, N,
        routing_weights.data_ptr() if N > 0 else None, wdt,
        expert_indices.data_ptr() if N > 0 else None, k, ctypes.byref(e),
        out.data_ptr() if N > 0 else None, _ptr(y) if N > 0 else None, counts.data_ptr(),
        offsets.data_ptr(), invalid.data_ptr(), workspace.data_ptr(), workspace.numel(),
        _stream(dev)), "yvmoe_dispatch")
    return out, counts, offsets, invalid, y


def moe_forward(x2d: torch.Tensor, router: RouterState, experts: PackedExperts,
                mix: Optional[torch.Tensor], skip: Optional[torch.Tensor],
                workspace: Optional[torch.Tensor] = None):
    """Whole layer. Returns (out [N,H], shared_out [N,H] or None, Routing)."""
    dev = _require_cuda(x2d, router.w_router, mix, skip, *experts.tensors())
    act = _act(x2d.dtype)
    N, H = x2d.shape
    if H != experts.hidden or H != router.hidden:
        raise ValueError(f"hidden size {H} does not match the layer ({experts.hidden})")
    E, k, S = router.num_experts, router.top_k, experts.num_shared
    routing = Routing.empty(N, E, k, dev)
    out = torch.empty_like(x2d)
    shared_out = torch.empty_like(x2d) if S > 0 else None
    need = workspace_bytes(N, act, router, experts)
    if workspace is None or workspace.numel() < need:
        workspace = _workspace(need, dev)
    if skip is not None and (skip.shape != x2d.shape or skip.dtype != x2d.dtype):
        raise ValueError("skip buffer must match x")
    if mix is not None and (mix.dtype != torch.float32 or mix.numel() != S):
        raise ValueError("mix must be fp32 [S]")
    r = router.struct()
    e = experts.struct()
    o = routing.struct()
    _lib.check(_lib.lib().yvmoe_forward(x2d.data_ptr(), act, N, ctypes.byref(r), ctypes.byref(e),
                                         _ptr(mix), _ptr(skip), out.data_ptr(), _ptr(shared_out),
                                         ctypes.byref(o), workspace.data_ptr(), workspace.numel(),
                                         _stream(dev)), "yvmoe_forward")
    return out, shared_out, routing


def moe_forward_static(x2d: torch.Tensor, router: RouterState, experts: PackedExperts,
                       mix: Optional[torch.Tensor], skip: Optional[torch.Tensor],
                       out: Optional[torch.Tensor] = None,
                       shared_out: Optional[torch.Tensor] = None,
                       routing: Optional[Routing] = None):
    """Whole layer on the library's own static scratch (yvmoe_forward_static): the library
    call allocates no device memory. Pass ``out``, ``shared_out`` and ``routing`` to make the
    whole call allocation-free (otherwise they are allocated here, before the library call).
    Calls that overlap on one GPU share its scratch and race. Returns (out, shared_out or
    None, Routing)."""
    dev = _require_cuda(x2d, router.w_router, mix, skip, out, shared_out, *experts.tensors())
    act = _act(x2d.dtype)
    N, H = x2d.shape
    if H != experts.hidden or H != router.hidden:
        raise ValueError(f"hidden size {H} does not match the layer ({experts.hidden})")
    E, k, S = router.num_experts, router.top_k, experts.num_shared
    if skip is not None and (skip.shape != x2d.shape or skip.dtype != x2d.dtype):
        raise ValueError("skip buffer must match x")
    if mix is not None and (mix.dtype != torch.float32 or mix.numel() != S):
        raise ValueError("mix must be fp32 [S]")
    if routing is None:
        routing = Routing.empty(N, E, k, dev)
    if out is None:
        out = torch.empty_like(x2d)
    if shared_out is None and S > 0:
        shared_out = torch.empty_like(x2d)
    for t in (out, shared_out):
        if t is not None and (t.shape != x2d.shape or t.dtype != x2d.dtype):
            raise ValueError("out and shared_out must match x")
    r = router.struct()
    e = experts.struct()
    o = routing.struct()
    _lib.check(_lib.lib().yvmoe_forward_static(x2d.data_ptr(), act, N, ctypes.byref(r),
                                                ctypes.byref(e), _ptr(mix), _ptr(skip),
                                                out.data_ptr(), _ptr(shared_out) if S > 0 else None,
                                                ctypes.byref(o), _stream(dev)),
               "yvmoe_forward_static")
    return out, (shared_out if S > 0 else None), routing


def few_workspace_bytes(n_tokens: int, act: int, top_k: int, experts: PackedExperts) -> int:
    """Workspace of moe_forward_few and experts_few (0 for sizes they do not take)."""
    return _few_workspace_bytes(n_tokens, act, top_k, experts.format, experts.num_routed, experts.num_shared,
                                experts.hidden, experts.ffn, experts.s_gate is not None)


@functools.lru_cache(maxsize=1024)
def _few_workspace_bytes(n_tokens, act, top_k, fmt, E, S, H, F, scales) -> int:
    p, s = 16, 16 if scales else None  # whether there are pointers, not which, goes into the size
    e = _lib.ExpertWeights(fmt, E, S, H, F, p, p, p, s, s, s)
    return int(_lib.lib().yvmoe_few_workspace_bytes(n_tokens, act, top_k, ctypes.byref(e)))


def _few_args(x2d, top_k, experts, mix, skip, workspace, dev):
    """Checks that the few-token calls share; returns (act, shared_out or None, workspace)."""
    act = _act(x2d.dtype)
    if x2d.dim() != 2 or x2d.shape[1] != experts.hidden:
        raise ValueError(f"x must be [N, {experts.hidden}], got {tuple(x2d.shape)}")
    N = x2d.shape[0]
    if N > _lib.FEW_TOKENS:
        raise ValueError(f"{N} tokens: the few-token layer takes up to {_lib.FEW_TOKENS} "
                         "(moe_forward and dispatch take any number)")
    if skip is not None and (skip.shape != x2d.shape or skip.dtype != x2d.dtype):
        raise ValueError("skip buffer must match x")
    if mix is not None and (mix.dtype != torch.float32 or mix.numel() != experts.num_shared):
        raise ValueError("mix must be fp32 [S]")
    if mix is None and experts.num_shared > 0:
        raise ValueError("shared experts need mix weights")
    need = few_workspace_bytes(N, act, top_k, experts)
    if workspace is None or workspace.numel() < need or workspace.device != dev:
        workspace = _workspace(need, dev)
    return act, (torch.empty_like(x2d) if experts.num_shared > 0 else None), workspace


def moe_forward_few(x2d: torch.Tensor, router: RouterState, experts: PackedExperts,
                    mix: Optional[torch.Tensor], skip: Optional[torch.Tensor],
                    workspace: Optional[torch.Tensor] = None):
    """moe_forward for up to 16 tokens in two kernels (yvmoe_forward_few), with fewer roundings:
    weights enter exactly, h keeps 16 bits, the outputs are rounded once. ``workspace`` is scratch of
    few_workspace_bytes (allocated here when None or too small); calls that overlap in time need
    one each. Returns (out [N,H], shared_out [N,H] or None, Routing)."""
    dev = _require_cuda(x2d, router.w_router, mix, skip, *experts.tensors())
    if router.hidden != experts.hidden or router.num_experts != experts.num_routed:
        raise ValueError("router and experts disagree")
    act, shared_out, workspace = _few_args(x2d, router.top_k, experts, mix, skip, workspace, dev)
    N = x2d.shape[0]
    routing = Routing.lazy(N, router.num_experts, router.top_k, dev)
    out = torch.empty_like(x2d)
    r, e, o = router.struct(), experts.struct(), routing.struct()
    _lib.check(_lib.lib().yvmoe_forward_few(
        x2d.data_ptr(), act, N, ctypes.byref(r), ctypes.byref(e), _ptr(mix), _ptr(skip), out.data_ptr(),
        _ptr(shared_out), ctypes.byref(o), workspace.data_ptr(), workspace.numel(), _stream(dev)),
        "yvmoe_forward_few")
    return out, shared_out, routing


def experts_few(x2d: torch.Tensor, routing_weights: torch.Tensor, expert_indices: torch.Tensor,
                experts: PackedExperts, mix: Optional[torch.Tensor] = None,
                skip: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None):
    """Routed and shared experts, weighted sum and skip residual of up to 16 tokens on a routing
    from any router (yvmoe_experts_few): ``routing_weights`` [N, k] fp32 or bf16,
    ``expert_indices`` [N, k] int64. Nothing synchronizes with the host. Returns (out [N,H],
    shared_out [N,H] or None, invalid [1] int32 = slots whose index lies outside [0, E), which
    add nothing)."""
    dev = _require_cuda(x2d, routing_weights, expert_indices, mix, skip, *experts.tensors())
    if expert_indices.dtype != torch.int64 or expert_indices.dim() != 2 or \
            expert_indices.shape[0] != x2d.shape[0]:
        raise ValueError("expert_indices must be int64 [N, k]")
    if routing_weights.shape != expert_indices.shape:
        raise ValueError(f"routing_weights must be {tuple(expert_indices.shape)}")
    k = expert_indices.shape[1]
    wdt = _act(routing_weights.dtype)
    act, shared_out, workspace = _few_args(x2d, k, experts, mix, skip, workspace, dev)
    out = torch.empty_like(x2d)
    invalid = torch.empty(1, dtype=torch.int32, device=dev)
    e = experts.struct()
    _lib.check(_lib.lib().yvmoe_experts_few(
        x2d.data_ptr(), act, x2d.shape[0], routing_weights.data_ptr(), wdt, expert_indices.data_ptr(), k,
        ctypes.byref(e), _ptr(mix), _ptr(skip), out.data_ptr(), _ptr(shared_out), invalid.data_ptr(),
        workspace.data_ptr(), workspace.numel(), _stream(dev)), "yvmoe_experts_few")
    return out, shared_out, invalid


@dataclass
class MoEGateState:
    """Device tensors and constants of one YvMoEGate, regrouped for yvmoe_moegate_logits."""

    num_experts: int
    hidden: int
    enc_dim: int
    dg_dim: int
    sparsity_k: int
    n_modalities: int
    heads: int                      # _lib.HEAD_* bits
    w_proj: torch.Tensor            # [(dg if HiCL) + Rh, H] activation dtype
    dg_bias: Optional[torch.Tensor]
    prototypes_t: Optional[torch.Tensor]
    eo_mat: Optional[torch.Tensor]  # [D, E] fp32
    modal_affinity: Optional[torch.Tensor]
    expert_bias: Optional[torch.Tensor]
    w_hicl: float
    w_got: float
    w_soft: float
    w_eo: float
    soft_temperature: float
    temperature: float
    soft_eps: float
    load_balance_alpha: float
    z_loss_alpha: float
    soft_budget: float
    capacity_loss: float

    def tensors(self):
        return [t for t in (self.w_proj, self.dg_bias, self.prototypes_t, self.eo_mat,
                            self.modal_affinity, self.expert_bias)
                if t is not None]

    def struct(self) -> _lib.MoEGate:
        return _lib.MoEGate(
            self.num_experts, self.hidden, self.enc_dim, self.dg_dim, self.sparsity_k,
            self.n_modalities, self.heads, 0, _ptr(self.w_proj), _ptr(self.dg_bias), _ptr(self.prototypes_t), _ptr(self.eo_mat),
            _ptr(self.modal_affinity), _ptr(self.expert_bias),
            self.w_hicl, self.w_got, self.w_soft, self.w_eo, self.soft_temperature,
            self.temperature, self.soft_eps, self.load_balance_alpha, self.z_loss_alpha,
            self.soft_budget, self.capacity_loss, 0.0)


def moegate_workspace_bytes(n_tokens: int, act: int, gate: MoEGateState) -> int:
    g = gate.struct()
    return int(_lib.lib().yvmoe_moegate_workspace_bytes(n_tokens, act, ctypes.byref(g)))


def moegate_logits(x2d: torch.Tensor, gate: MoEGateState, modal_id: Optional[torch.Tensor] = None,
                   workspace: Optional[torch.Tensor] = None):
    """YvMoEGate logits [N, E] fp32 (temperature-scaled) and the routing loss [1] fp32."""
    dev = _require_cuda(x2d, modal_id, *gate.tensors())
    act = _act(x2d.dtype)
    N, H = x2d.shape
    if H != gate.hidden:
        raise ValueError(f"hidden size {H} does not match the gate ({gate.hidden})")
    if modal_id is not None and (modal_id.dtype != torch.int32 or modal_id.numel() != N):
        raise ValueError("modal_id must be int32 [N]")
    E = gate.num_experts
    logits = torch.empty(N, E, dtype=torch.float32, device=dev)
    loss = torch.empty(1, dtype=torch.float32, device=dev)
    need = moegate_workspace_bytes(N, act, gate)
    if need == 0:
        raise ValueError("yvmoe_moegate_workspace_bytes rejected the gate state")
    if workspace is None or workspace.numel() < need:
        workspace = _workspace(need, dev)
    g = gate.struct()
    _lib.check(_lib.lib().yvmoe_moegate_logits(x2d.data_ptr() if N > 0 else None, act, N,
                                                ctypes.byref(g), _ptr(modal_id),
                                                logits.data_ptr() if N > 0 else None,
                                                loss.data_ptr(), workspace.data_ptr(),
                                                workspace.numel(), _stream(dev)),
               "yvmoe_moegate_logits")
    return logits, loss


def moegate_forward(x2d: torch.Tensor, gate: MoEGateState, top_k: int,
                    modal_id: Optional[torch.Tensor] = None,
                    workspace: Optional[torch.Tensor] = None):
    """YvMoEGate logits [N, E], loss [1] and the fixed-mode routing, in one library call.

    Returns (logits, loss, Routing, workspace); the routing can be passed on to expert_ffn.
    """
    dev = _require_cuda(x2d, modal_id, *gate.tensors())
    act = _act(x2d.dtype)
    N, H = x2d.shape
    if H != gate.hidden:
        raise ValueError(f"hidden size {H} does not match the gate ({gate.hidden})")
    if modal_id is not None and (modal_id.dtype != torch.int32 or modal_id.numel() != N):
        raise ValueError("modal_id must be int32 [N]")
    E = gate.num_experts
    g = gate.struct()
    need = int(_lib.lib().yvmoe_moegate_forward_workspace_bytes(N, act, top_k, ctypes.byref(g)))
    if need == 0:
        raise ValueError("yvmoe_moegate_forward_workspace_bytes rejected the gate state / top_k")
    if workspace is None or workspace.numel() < need:
        workspace = _workspace(need, dev)
    logits = torch.empty(N, E, dtype=torch.float32, device=dev)
    loss = torch.empty(1, dtype=torch.float32, device=dev)
    routing = Routing.empty(N, E, top_k, dev)
    o = routing.struct()
    _lib.check(_lib.lib().yvmoe_moegate_forward(x2d.data_ptr() if N > 0 else None, act, N,
                                                 ctypes.byref(g), _ptr(modal_id), top_k,
                                                 logits.data_ptr() if N > 0 else None,
                                                 loss.data_ptr(), ctypes.byref(o),
                                                 workspace.data_ptr(), workspace.numel(),
                                                 _stream(dev)), "yvmoe_moegate_forward")
    return logits, loss, routing, workspace


def moe_forward_moegate(x2d: torch.Tensor, gate: MoEGateState, top_k: int, experts: PackedExperts,
                        mix: Optional[torch.Tensor], skip: Optional[torch.Tensor],
                        modal_id: Optional[torch.Tensor] = None,
                        route_logits: Optional[torch.Tensor] = None,
                        workspace: Optional[torch.Tensor] = None):
    """Whole layer with a YvMoEGate router. Returns (out, shared_out or None, Routing, logits,
    loss, workspace); ``route_logits`` (fp32 [N, E]) routes on earlier logits instead."""
    dev = _require_cuda(x2d, mix, skip, modal_id, route_logits, *gate.tensors(), *experts.tensors())
    act = _act(x2d.dtype)
    N, H = x2d.shape
    if H != experts.hidden or H != gate.hidden:
        raise ValueError(f"hidden size {H} does not match the layer ({experts.hidden})")
    if skip is not None and (skip.shape != x2d.shape or skip.dtype != x2d.dtype):
        raise ValueError("skip buffer must match x")
    if mix is not None and (mix.dtype != torch.float32 or mix.numel() != experts.num_shared):
        raise ValueError("mix must be fp32 [S]")
    if modal_id is not None and (modal_id.dtype != torch.int32 or modal_id.numel() != N):
        raise ValueError("modal_id must be int32 [N]")
    E, S = gate.num_experts, experts.num_shared
    if route_logits is not None and (route_logits.dtype != torch.float32 or
                                     tuple(route_logits.shape) != (N, E)):
        raise ValueError("route_logits must be fp32 [N, E]")
    g = gate.struct()
    e = experts.struct()
    need = int(_lib.lib().yvmoe_forward_moegate_workspace_bytes(N, act, top_k, ctypes.byref(g),
                                                                ctypes.byref(e)))
    if need == 0:
        raise ValueError("yvmoe_forward_moegate_workspace_bytes rejected the gate / experts / top_k")
    if workspace is None or workspace.numel() < need:
        workspace = _workspace(need, dev)
    routing = Routing.empty(N, E, top_k, dev)
    out = torch.empty_like(x2d)
    shared_out = torch.empty_like(x2d) if S > 0 else None
    logits = torch.empty(N, E, dtype=torch.float32, device=dev)
    loss = torch.empty(1, dtype=torch.float32, device=dev)
    o = routing.struct()
    _lib.check(_lib.lib().yvmoe_forward_moegate(
        x2d.data_ptr() if N > 0 else None, act, N, ctypes.byref(g), _ptr(modal_id), top_k,
        _ptr(route_logits), ctypes.byref(e), _ptr(mix), _ptr(skip),
        out.data_ptr() if N > 0 else None, _ptr(shared_out) if N > 0 else None, ctypes.byref(o),
        logits.data_ptr() if N > 0 else None, loss.data_ptr(), workspace.data_ptr(),
        workspace.numel(), _stream(dev)), "yvmoe_forward_moegate")
    return out, shared_out, routing, logits, loss, workspace


_RMS_PARAMS1, _RMS_PARAMS2 = _lib.RMSNormParams * 1, _lib.RMSNormParams * 2


def rms_norm(x: torch.Tensor, norms, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """RMSNorm over the last dimension, one or two norms in sequence in one pass.

    ``norms`` is a sequence of (weight, bias or None, eps); two entries apply the second norm to
    the first one's output rounded to x's dtype (YvHybridBlock's norm_fusion then norm_mlp,
    model/core/hybrid.py:1359, :1310). Each norm follows fused_rms_norm
    (opss/kernels/fused_rms_norm.py:42): fp32 sum of squares, (x / sqrt(Σx²/H + eps)) * weight
    rounded once, + bias rounded again (model/core/norms.py:998-999). ``out`` may be x.
    """
    norms = tuple(norms)
    if len(norms) not in (1, 2):
        raise ValueError("rms_norm takes one or two norms")
    shape, dt = x.shape, x.dtype
    H = shape[-1]
    dev = _require_cuda(x, *norms[0][:2], *norms[-1][:2], out)
    act = _act(dt)
    params = (_RMS_PARAMS1 if len(norms) == 1 else _RMS_PARAMS2)()
    for p, (w, b, eps) in zip(params, norms):
        if w.dtype != dt or w.numel() != H or (b is not None and (b.dtype != dt or b.numel() != H)):
            raise ValueError(f"norm weight/bias must be {dt} [{H}]")
        p.weight = w.data_ptr()
        p.bias = None if b is None else b.data_ptr()
        p.eps = float(eps)
    if out is None:
        out = torch.empty_like(x)
    elif out.shape != shape or out.dtype != dt:
        raise ValueError("out must match x")
    N = x.numel() // H if H else 0
    rc = _lib.lib().yvmoe_rmsnorm(x.data_ptr() if N > 0 else None, act, N, H, params, len(norms),
                                  out.data_ptr() if N > 0 else None, _stream(dev))
    if rc:
        _lib.check(rc, "yvmoe_rmsnorm")
    return out


def int4_linear(x: torch.Tensor, weight: PackedLinear, bias: Optional[torch.Tensor] = None,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x [..., in] · Wᵀ (+ bias [out]) with a 4-bit weight (quant.pack_linear), in fp32 sums of exact
    products rounded once to x's dtype (bf16 or fp32), which bias and ``out`` share. Up to 2^30
    rows; ``out`` [..., out] must not overlap x or the weight, nor bias unless it is bias, of one row. An
    infinity or NaN in a row of x makes all its outputs NaN."""
    K, O = weight.in_features, weight.out_features
    shape, dt = x.shape, x.dtype
    if x.dim() == 0 or shape[-1] != K:
        raise ValueError(f"x must be [..., {K}], got {tuple(shape)}")
    rows = x.numel() // K
    if rows > 1 << 30:
        raise ValueError(f"{rows} rows: a call takes up to 2^30")
    dev = _require_cuda(x, weight.codes, weight.scales, bias, out)
    act = _act(dt)
    if bias is not None and (bias.dtype != dt or bias.numel() != O):
        raise ValueError(f"bias must be {dt} [{O}]")
    want = (*shape[:-1], O)
    if out is None:
        out = torch.empty(want, dtype=dt, device=x.device)
    elif out.shape != want or out.dtype != dt:
        raise ValueError(f"out must be {dt} {tuple(want)}")
    w = weight.struct()
    rc = _lib.lib().yvmoe_int4_linear(x.data_ptr(), act, rows, ctypes.byref(w), _ptr(bias),
                                      out.data_ptr(), _stream(dev))
    if rc:
        _lib.check(rc, "yvmoe_int4_linear")
    return out


# ---------------------------------------------------------------- 8-bit floating point
def _launch(dev: torch.device, entry, *args) -> int:
    """Calls an entry of the library with ``dev`` as the current device."""
    if torch._C._cuda_getDevice() == dev.index:
        return entry(*args)
    with torch.cuda.device(dev):
        return entry(*args)


def _same_device(*ts: Optional[torch.Tensor]) -> torch.device:
    """_require_cuda, on one device."""
    dev = None
    for t in ts:
        if t is None:
            continue
        if dev is None:
            dev = t.device
            if dev.type != "cuda":
                raise ValueError("libyvmoe computes on the GPU only: got a CPU tensor")
        elif t.device != dev:
            raise ValueError(f"tensors on {t.device} and {dev}")
        if not t.is_contiguous():
            raise ValueError("libyvmoe needs contiguous tensors")
    return dev


_MAX_ROWS, _MAX_FEATURES = 1 << 24, 1 << 20  # of a call; the library's counts have 32 bits


def _too_large(rows: int, *features: int) -> None:
    if rows > _MAX_ROWS:
        raise ValueError(f"{rows} rows: a call takes up to 2^24")
    raise ValueError(f"{max(features)} features: a call takes up to 2^20")


def _no_tangents(what: str, *ts: Optional[torch.Tensor]) -> None:
    for t in ts:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{what} has no forward-mode derivative")


def _no_gradients(what: str, *ts: Optional[torch.Tensor]) -> None:
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                raise NotImplementedError(f"{what} is inference only: an operand requires a gradient (detach it, or use "
                                          "torch.no_grad)")
    if forward_ad._current_level >= 0:
        _no_tangents(what, *ts)


def quantize_fp8_rows(x: torch.Tensor) -> Fp8Rows:
    """Rows of x [..., features] (bf16 or fp32) in e4m3fn with a scale per 128 values, the left operand of
    fp8_linear: scale = max(max|x| / 448, 1e-12), code = e4m3fn(x / scale), in fp32 divisions and rounded to
    nearest even (quantize_to_fp8, opss/quantize/engine.py:841-883, per 128 values). A group with an infinity or
    NaN makes every product of its row NaN. Up to 2^24 rows of up to 2^20 features; inference only."""
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"x must be [..., features], got {tuple(x.shape)}")
    if x.requires_grad or forward_ad._current_level >= 0:
        _no_gradients("quantize_fp8_rows", x)
    K = x.shape[-1]
    N, groups = x.numel() // K, -(-K // 128)
    if N > _MAX_ROWS or K > _MAX_FEATURES:
        _too_large(N, K)
    dev, act = _same_device(x), _act(x.dtype)
    rows = Fp8Rows(K, torch.empty(N, groups * 128, dtype=torch.float8_e4m3fn, device=dev),
                   torch.empty(groups, N, dtype=torch.float32, device=dev))
    rc = _launch(dev, _lib.lib().yvmoe_quantize_fp8_rows, x.data_ptr(), act, N, K, rows.codes.data_ptr(),
                 rows.scales.data_ptr(), _stream(dev))
    if rc:
        _lib.check(rc, "yvmoe_quantize_fp8_rows")
    return rows


def _fp8_out(out: Optional[torch.Tensor], shape, dev) -> torch.Tensor:
    if out is None:
        return torch.empty(shape, dtype=torch.bfloat16, device=dev)
    if tuple(out.shape) != tuple(shape) or out.dtype != torch.bfloat16:
        raise ValueError(f"out must be bfloat16 {tuple(shape)}")
    return out


def fp8_linear(x, weight: PackedFp8Linear, bias: Optional[torch.Tensor] = None,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x · Wᵀ (+ bias [out] bf16) with both operands in 8-bit floating point: W in e4m3fn with a scale per
    128 x 128 block (quant.pack_fp8_linear), x [..., in] bf16, rounded to e4m3fn with a scale per 128 values in
    the call, or rows that are already (Fp8Rows). fp32 sums, rounded once to bf16 [..., out]; the matrix unit
    keeps about 16 bits of a block's sum, so there are no fp32 outputs. Up to 2^24 rows; inference only.
    ``out`` must overlap no input."""
    K, O = weight.in_features, weight.out_features
    rows = isinstance(x, Fp8Rows)
    if rows:
        if x.features != K:
            raise ValueError(f"rows have {x.features} features, the weight {K}")
        _no_gradients("fp8_linear", x.codes, x.scales, weight.scales, bias, out)
        N = x.codes.shape[0]
        if N > _MAX_ROWS or K > _MAX_FEATURES or O > _MAX_FEATURES:
            _too_large(N, K, O)
        lead, dev = (N,), _same_device(x.codes, x.scales, weight.codes, weight.scales, bias, out)
    else:
        if x.dim() == 0 or x.shape[-1] != K:
            raise ValueError(f"x must be [..., {K}], got {tuple(x.shape)}")
        if x.dtype != torch.bfloat16:
            raise ValueError(f"x must be bfloat16 or Fp8Rows, got {x.dtype}")
        _no_gradients("fp8_linear", x, weight.scales, bias, out)
        N = x.numel() // K
        if N > _MAX_ROWS or K > _MAX_FEATURES or O > _MAX_FEATURES:
            _too_large(N, K, O)
        lead, dev = x.shape[:-1], _same_device(x, weight.codes, weight.scales, bias, out)
    if bias is not None and (bias.dtype != torch.bfloat16 or bias.numel() != O):
        raise ValueError(f"bias must be bfloat16 [{O}]")
    out = _fp8_out(out, (*lead, O), dev)
    l, w = _lib.lib(), weight.struct()
    need = l.yvmoe_fp8_linear_rows_workspace_bytes if rows else l.yvmoe_fp8_linear_workspace_bytes
    nbytes = need(N, K, O)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    tail = (N, ctypes.byref(w), _ptr(bias), out.data_ptr(), ws.data_ptr(), nbytes, _stream(dev))
    if rows:
        rc = _launch(dev, l.yvmoe_fp8_linear_rows, x.codes.data_ptr(), x.scales.data_ptr(), *tail)
    else:
        rc = _launch(dev, l.yvmoe_fp8_linear, x.data_ptr(), *tail)
    if rc:
        _lib.check(rc, "yvmoe_fp8_linear")
    return out


def fp8_swiglu(x: torch.Tensor, gate: PackedFp8Linear, up: PackedFp8Linear, down: PackedFp8Linear,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The gated feed-forward block (:func:`swiglu`) on 8-bit weights: products as in :func:`fp8_linear`, the
    activated product in fp32 and rounded to e4m3fn with a scale per 128 values. x [..., H] and the result
    bf16, gate and up F x H, down H x F. Inference only. ``out`` must overlap no input."""
    H, F = gate.in_features, gate.out_features
    if (up.in_features, up.out_features, down.in_features, down.out_features) != (H, F, F, H):
        raise ValueError(f"gate {F} x {H}, up {up.out_features} x {up.in_features}, down {down.out_features} x "
                         f"{down.in_features} are no gated block")
    if x.dim() == 0 or x.shape[-1] != H:
        raise ValueError(f"x must be [..., {H}], got {tuple(x.shape)}")
    if x.dtype != torch.bfloat16:
        raise ValueError(f"x must be bfloat16, got {x.dtype}")
    _no_gradients("fp8_swiglu", x, gate.scales, up.scales, down.scales, out)
    N = x.numel() // H
    if N > _MAX_ROWS or H > _MAX_FEATURES or F > _MAX_FEATURES:
        _too_large(N, H, F)
    dev = _same_device(x, gate.codes, gate.scales, up.codes, up.scales, down.codes, down.scales, out)
    out = _fp8_out(out, x.shape, dev)
    l = _lib.lib()
    g, u, d = gate.struct(), up.struct(), down.struct()
    nbytes = l.yvmoe_fp8_swiglu_workspace_bytes(N, H, F)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    rc = _launch(dev, l.yvmoe_fp8_swiglu, x.data_ptr(), N, ctypes.byref(g), ctypes.byref(u), ctypes.byref(d),
                 out.data_ptr(), ws.data_ptr(), nbytes, _stream(dev))
    if rc:
        _lib.check(rc, "yvmoe_fp8_swiglu")
    return out


# ---------------------------------------------------------------- gated feed-forward block
def _aligned(t: torch.Tensor) -> torch.Tensor:
    """``t`` at a 16-byte address (a copy where a view starts elsewhere)."""
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _swiglu_forward(x2d, w_gate, w_up, w_down, keep: bool):
    """(out, what the backward pass needs or None) of rows [N, H]."""
    l, (N, H), F, dt, dev = _lib.lib(), x2d.shape, w_gate.shape[0], x2d.dtype, x2d.device
    act = _act(dt)
    out = torch.empty_like(x2d)
    w = _lib.SwiGLUWeights(H, F, w_gate.data_ptr(), w_up.data_ptr(), w_down.data_ptr())
    nbytes = l.yvmoe_swiglu_workspace_bytes(N, act, H, F, 0)
    if nbytes == 0 and N > 0:
        raise ValueError(f"swiglu: {l.yvmoe_last_error().decode(errors='replace')}")
    saved = torch.empty(l.yvmoe_swiglu_saved_bytes(N, F) // 4, dtype=torch.float32, device=dev) if keep else None
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    rc = _launch(dev, l.yvmoe_swiglu_forward, x2d.data_ptr(), act, N, ctypes.byref(w), _ptr(saved), out.data_ptr(),
                 ws.data_ptr(), nbytes, _stream(dev))
    if rc:
        _lib.check(rc, "yvmoe_swiglu_forward")
    return out, saved


_training = weakref.WeakSet()  # contexts of swiglu calls whose graphs live
_training_lock = threading.Lock()  # one thread's call is added while another's backward pass looks through them


def _leaves(ctx) -> set:
    """ids of the leaves that a backward pass through a call adds gradients to: its own (ctx.leaves), and those behind
    views, casts, copies and the layers before it. A graph keeps its leaves, so an id stands for one tensor."""
    found, seen, todo = set(ctx.leaves), set(), [ctx]
    while todo:
        for node, _ in getattr(todo.pop(), "next_functions", ()):
            if node is None or node in seen:
                continue
            seen.add(node)
            if node.name() == "torch::autograd::AccumulateGrad":
                found.add(id(node.variable))
            else:
                todo.append(node)
    return found


def _refuse_other_streams(ctx) -> None:
    """A leaf's gradient is added on the stream of its oldest living graph. Where that is not the stream that is being
    captured, torch has the two wait for one another, which a capture does not survive. Only graphs with a swiglu call in
    them are known here."""
    with _training_lock:
        others = [other for other in _training if other.stream != ctx.stream]
    if not others:
        return
    mine = _leaves(ctx)
    for other in others:
        if not mine.isdisjoint(_leaves(other)):
            raise RuntimeError("swiglu: this backward pass is being captured while a graph of the same leaves that was "
                               "recorded on another stream lives: drop its outputs first")


class _SwiGLU(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x2d, w_gate, w_up, w_down):
        out, saved = _swiglu_forward(x2d, w_gate, w_up, w_down, True)
        ctx.save_for_backward(x2d, w_gate, w_up, w_down, saved)
        ctx.stream = _stream(x2d.device)
        # x2d may be a view of the leaf
        leaves = (t if t.is_leaf else t._base for t in (x2d, w_gate, w_up, w_down))
        ctx.leaves = {id(t) for t in leaves if t is not None and t.is_leaf and t.requires_grad}
        with _training_lock:
            _training.add(ctx)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        if torch.cuda.is_current_stream_capturing():
            _refuse_other_streams(ctx)
        x, wg, wu, wd, saved = ctx.saved_tensors
        l, (N, H), F, dev = _lib.lib(), x.shape, wg.shape[0], x.device
        act = _act(x.dtype)
        dy = _aligned(dy.contiguous())
        grads = [torch.empty_like(t) if need else None
                 for t, need in zip((x, wg, wu, wd), ctx.needs_input_grad)]
        w = _lib.SwiGLUWeights(H, F, wg.data_ptr(), wu.data_ptr(), wd.data_ptr())
        nbytes = l.yvmoe_swiglu_workspace_bytes(N, act, H, F, 1)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        rc = _launch(dev, l.yvmoe_swiglu_backward, dy.data_ptr(), x.data_ptr(), saved.data_ptr(), act, N,
                     ctypes.byref(w), *map(_ptr, grads), ws.data_ptr(), nbytes, _stream(dev))
        if rc:
            _lib.check(rc, "yvmoe_swiglu_backward")
        return tuple(grads)


def swiglu(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor) -> torch.Tensor:
    """The gated feed-forward block of one dense expert (YvSwiGLUExpert.forward,
    model/moe/expert.py:475-489): (silu(x w_gateᵀ) · (x w_upᵀ)) w_downᵀ, with gradients of x and the weights.

    x [..., H], w_gate and w_up [F, H], w_down [H, F] (nn.Linear.weight), all bf16 or all fp32, contiguous;
    any sizes up to 2^24 rows and 2^20 features. Sums are fp32; bf16 rounds the activated product and the two
    gradients before it once each, as operands, and the outputs. For the backward pass the call keeps x and the
    two projections in fp32 (8 bytes a row and feature of F). The gradients are not differentiable again, and there
    are no forward-mode derivatives. A backward pass that is being captured is refused while another
    call's graph with some of the same leaves (weights or inputs, also behind other operations) that was recorded on
    another stream lives; leaves that are shared with a graph without such a call are not seen.
    """
    if w_gate.dim() != 2 or w_up.shape != w_gate.shape or w_down.shape != w_gate.shape[::-1]:
        raise ValueError(f"weights must be [F, H], [F, H], [H, F], got {tuple(w_gate.shape)}, "
                         f"{tuple(w_up.shape)}, {tuple(w_down.shape)}")
    F, H = w_gate.shape
    if F < 1 or H < 1:
        raise ValueError(f"a gated block needs features, got hidden {H}, ffn {F}")
    if x.dim() == 0 or x.shape[-1] != H:
        raise ValueError(f"x must be [..., {H}], got {tuple(x.shape)}")
    if not (x.dtype == w_gate.dtype == w_up.dtype == w_down.dtype):
        raise ValueError(f"x and the weights must have one dtype, got {x.dtype}, {w_gate.dtype}, {w_up.dtype}, "
                         f"{w_down.dtype}")
    _act(x.dtype)
    N = x.numel() // H
    if N > _MAX_ROWS or H > _MAX_FEATURES or F > _MAX_FEATURES:
        _too_large(N, H, F)
    if forward_ad._current_level >= 0:
        _no_tangents("swiglu", x, w_gate, w_up, w_down)
    _same_device(x, w_gate, w_up, w_down)
    x2d = _aligned(x if x.dim() == 2 else x.view(-1, H))
    w_gate, w_up, w_down = _aligned(w_gate), _aligned(w_up), _aligned(w_down)
    if torch.is_grad_enabled() and (x.requires_grad or w_gate.requires_grad or w_up.requires_grad
                                    or w_down.requires_grad):
        out = _SwiGLU.apply(x2d, w_gate, w_up, w_down)
    else:
        out, _ = _swiglu_forward(x2d, w_gate, w_up, w_down, False)
    return out if x.dim() == 2 else out.view(x.shape)
