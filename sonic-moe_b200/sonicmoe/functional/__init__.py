"""Functional API of the reference (``sonicmoe/functional/__init__.py``), on the FP8 B200 engine.

Same names, arguments and return values as the reference:

* ``moe_TC_softmax_topk_layer`` (reference ``functional/__init__.py:482-557``)
* ``moe_general_routing_inputs`` (reference ``functional/__init__.py:571-652``)
* ``TC_topk_router_metadata_triton`` / ``general_routing_router_metadata_triton`` and
  ``_topk_softmax_fwd`` (reference ``triton_kernels/__init__.py:78-146, 281-353``,
  ``forward.py:107-141``), here backed by the CUDA metadata and router kernels.

Weight-format contract (reference ``functional/__init__.py:560-566``): ``w1`` is the
``(2I, H, E)`` view of ``c_fc.weight`` ``[E, 2I, H]`` (stride order (2, 0, 1)), interleaved
``[g0, u0, g1, u1, ...]`` or, with ``concat_layout=True``, ``[g0..g_{I-1}, u0..u_{I-1}]``;
``w2`` is the ``(H, I, E)`` view of ``c_proj.weight`` ``[E, H, I]``.  The bf16 weights are
quantised to e4m3 with 128x128 UE8M0 block scales on first use and cached per weight version;
already prepared :class:`~sonicmoe.ops.Fp8ExpertWeights` may be passed instead, or for inference
:class:`~sonicmoe.ops.Int4ExpertWeights` (``prepare_int4_weights``: 4-bit codes with group scales, x
kept in bf16; decoding is bound by the weights' bytes).

Op boundary: as in the reference, the router top-k (``sonicmoe::_topk_fwd``,
``sonicmoe::_softmax_topk_fwd``, in ``forward.py``) and the routing metadata
(``triton_kernels::TC_topk_router_metadata``, ``triton_kernels::general_routing_router_metadata``)
are ``torch.library.custom_op``s writing into caller-allocated outputs; the engine's layer forward
after the router GEMM is one more registered op per entry point (``sonicmoe::fp8_moe_tc_forward``,
``sonicmoe::fp8_moe_general_forward``, with fake implementations for tracing; the like for 4-bit weights), so
``torch.compile`` traces a whole ``MoE`` forward without a graph break.

Training: with ``is_inference_mode_enabled=False`` while autograd is recording and an input or
weight requires grad, ``moe_TC_softmax_topk_layer`` and ``moe_general_routing_inputs`` run the
training forward (the up GEMM also stores the pre-activation h) inside an autograd function whose
backward is the engine's FP8 backward (``ops.moe_backward``: dx, the router logits' or router
scores' gradient, dw1, dw2), as the reference's ``_UpProjection`` / ``_DownProjection`` / router
functions do.

Differences from the reference, all explicit errors: biases and activations other than SwiGLU
raise ``NotImplementedError`` (the FP8 engine implements the bias-free SwiGLU layer); the backward
covers ``moe_TC_softmax_topk_layer`` and ``moe_general_routing_inputs`` (both w1 layouts,
I % 256 == 0) -- the fused router and prepared e4m3 weights raise ``NotImplementedError`` when a
gradient is requested, instead of returning an output whose weights would never receive one.
"""
import itertools
import weakref

import torch
import torch.autograd.forward_ad as fwAD
import torch.nn.functional as F
from torch.multiprocessing.reductions import StorageWeakRef

from .. import ops
from ..enums import ActivationType
from ..ops import Fp8ExpertWeights, Int4ExpertWeights
from .forward import _topk_fwd, _topk_softmax_fwd  # noqa: F401  (registers the router ops)

__all__ = [
    "moe_TC_softmax_topk_layer",
    "moe_general_routing_inputs",
    "TC_topk_router_metadata_triton",
    "general_routing_router_metadata_triton",
    "prepare_fp8_weights",
    "prepare_int4_weights",
    "switch_load_balancing_loss",
    "Fp8ExpertWeights",
    "Int4ExpertWeights",
]

# Prepared FP8 weights, per tensor that owns the weight's storage (the root of its view chain):
# id(owner) -> (weak reference to owner, {layout: (state, prepared)}).  An entry is dropped when its
# tensor is freed, so a new weight tensor that happens to be allocated at a freed one's address can
# never see the old tensor's FP8 copy.  (Tensors cannot be weak dictionary keys: their == is
# elementwise.)
_WEIGHT_CACHE: dict = {}


def _forget(key: int, ref) -> None:
    entry = _WEIGHT_CACHE.get(key)
    if entry is not None and entry[0] is ref:
        del _WEIGHT_CACHE[key]


def _as_expert_major(w: torch.Tensor) -> torch.Tensor:
    """(N, K, E) reference view -> [E, N, K] tensor (a view when w came from permute(1, 2, 0))."""
    return w.permute(2, 0, 1)


def _storage_owner(t: torch.Tensor) -> torch.Tensor:
    while t._base is not None:
        t = t._base
    return t


def prepare_fp8_weights(w, concat_glu: bool = False, with_t: bool = False) -> Fp8ExpertWeights:
    """e4m3 + 128x128 UE8M0 version of an expert weight given in the reference's (N, K, E) view.

    Cached on the tensor that owns the weight's storage, for its current (data pointer, version
    counter, shape, strides, layout): repeated forwards with unchanged weights quantise once, an
    in-place update or a storage swap re-quantises, and the entry is dropped with the tensor.
    with_t (training): the result also holds the transposed copy the backward reads (prepared in the
    same pass over the weight, or added to a cached entry that lacks it).
    """
    if isinstance(w, Fp8ExpertWeights):
        return w
    owner = _storage_owner(w)
    layout = (tuple(w.shape), tuple(w.stride()), bool(concat_glu), w.dtype)
    state = (w.data_ptr(), w._version)
    entry = _WEIGHT_CACHE.get(id(owner))
    per_owner = entry[1] if entry is not None and entry[0]() is owner else None
    if per_owner is not None:
        hit = per_owner.get(layout)
        if hit is not None and hit[0] == state:
            if with_t and hit[1].t is None:
                hit[1].t = ops.weight_prep_t(hit[1])
            return hit[1]
    with torch.no_grad():
        prepared = ops.weight_prep(_as_expert_major(w.detach()), concat_glu=concat_glu, with_t=with_t)
    if per_owner is None:
        key = id(owner)
        ref = weakref.ref(owner, lambda r, k=key: _forget(k, r))
        per_owner = {}
        _WEIGHT_CACHE[key] = (ref, per_owner)
    per_owner[layout] = (state, prepared)  # only the newest version of each layout is kept
    return prepared


def prepare_int4_weights(w: torch.Tensor, group_size: int = 128, concat_glu: bool = False,
                         out: Int4ExpertWeights | None = None) -> Int4ExpertWeights:
    """4-bit version, with a scale per ``group_size`` (32, 64 or 128) input columns, of an expert weight
    given in the reference's (N, K, E) view.  Nothing is cached: the caller keeps the result.  ``out``: an
    earlier result of the same shape, group and layout, whose buffers are written again."""
    with torch.no_grad():
        return ops.weight_prep_int4(_as_expert_major(w.detach()), group_size, concat_glu=concat_glu, out=out)


class Int4Copies:
    """4-bit copies of a module's expert weights w1 [E, 2I, H] and w2 [E, H, I], made again when a weight has changed:
    another storage, address, shape or version counter (inference tensors have no counter, so there only the former).

    Weights that were put away (None, empty, or on another kind of device than the copies) leave the copies in use,
    unless they were changed first.  A deep or pickled copy of this object belongs to other weights and makes its own
    at the first use.

    New copies go into the old ones' buffers, which a captured graph may still read, and are complete on every stream
    when they are given out (the device is waited for before and after).  A capture that finds a weight changed records
    the preparation, of copies of its own."""

    _known = weakref.WeakValueDictionary()  # for traced callers, which name it by its number
    _numbers = itertools.count()

    def __init__(self, group_size: int, copies=(None, None)):
        self.group_size = group_size
        # the copies and the states of the weights they were made from: one value, so that a thread never sees the
        # one without the other
        self._now = tuple(copies), (None, None)
        # apart from the copies themselves, which a traced caller must not depend on: they may be made again
        self._on = None if copies[0] is None else copies[0].q.device.type
        self.handle = next(self._numbers)
        self._known[self.handle] = self

    @property
    def copies(self):
        return self._now[0]

    def __reduce__(self):
        return Int4Copies, (self.group_size, self.copies)

    @staticmethod
    def _state(w):
        storage = w.untyped_storage()
        # the weak reference keeps a freed storage's identity from being given to another
        return StorageWeakRef(storage), storage._cdata, w.data_ptr(), w.shape, w.dtype, \
            None if w.is_inference() else w._version

    def away(self, w1, w2) -> bool:
        """A weight cannot be prepared, and there are copies to go on with."""
        return self._on is not None and any(w is None or w.numel() == 0 or w.device.type != self._on for w in (w1, w2))

    def current(self, w1, w2, again: bool = False):
        """The copies (w1's, w2's) of the weights as they are; again: made again in any case."""
        weights, (copies, states) = (w1, w2), self._now
        if self.away(w1, w2):
            for w, state in zip(weights, states):
                if w is not None and state is not None and not w.is_inference() and (state[-1] or 0) < w._version:
                    raise RuntimeError("the expert weights were changed and put away since their 4-bit copies were made: "
                                       "bring them back, or call use_int4_experts with them in place")
            return copies
        fresh = [not again and self._fresh(w, s) for w, s in zip(weights, states)]
        return copies if all(fresh) else self._make(weights, copies, fresh)

    def _make(self, weights, copies, fresh):
        cuda = all(w.is_cuda for w in weights)
        if cuda and torch.cuda.is_current_stream_capturing():  # nothing to keep of launches that have not run
            return tuple(c if ok else prepare_int4_weights(w.permute(1, 2, 0), self.group_size)
                         for w, c, ok in zip(weights, copies, fresh))
        if cuda:
            torch.cuda.synchronize(weights[0].device)
        states = tuple(self._state(w) for w in weights)
        self._now = copies, (None, None)
        made = tuple(c if ok else prepare_int4_weights(
            w.permute(1, 2, 0), self.group_size,
            out=c if c is not None and c.shape == tuple(w.shape) and c.q.device == w.device else None)
            for w, c, ok in zip(weights, copies, fresh))
        if cuda:
            torch.cuda.synchronize(weights[0].device)
        self._now, self._on = (made, states), made[0].q.device.type
        return made

    def _fresh(self, w, state):
        if state is None:
            return False
        _, storage, ptr, shape, dtype, version = state
        return (w.data_ptr() == ptr and (w.is_inference() or w._version == version)
                and w.untyped_storage()._cdata == storage and w.shape == shape and w.dtype == dtype)


def _int4_pair(w1, w2, concat_layout) -> bool:
    """True for 4-bit expert weights (both must be, and w1 prepared for concat_layout)."""
    if not (isinstance(w1, Int4ExpertWeights) or isinstance(w2, Int4ExpertWeights)):
        return False
    if not (isinstance(w1, Int4ExpertWeights) and isinstance(w2, Int4ExpertWeights)):
        raise ValueError("w1 and w2 must both be 4-bit expert weights")
    if w1.concat_glu != bool(concat_layout):
        raise ValueError("prepared w1 layout does not match concat_layout")
    return True


def _prepared(w) -> bool:
    return isinstance(w, (Fp8ExpertWeights, Int4ExpertWeights))


def _check_common(b1, b2, activation_type):
    assert ((b1 is None) and (b2 is None)) or (
        (b1 is not None) and (b2 is not None)
    ), "b1 and b2 has to be None or not None at the same time!"
    if b1 is not None:
        raise NotImplementedError("the FP8 engine implements the bias-free layer (b1 = b2 = None)")
    if isinstance(activation_type, str):
        activation_type = ActivationType(activation_type)
    if activation_type != ActivationType.SWIGLU:
        raise NotImplementedError(f"the FP8 engine implements SwiGLU only, got {activation_type}")
    return activation_type


def _wants_training(is_inference_mode_enabled, *tensors) -> bool:
    """True when autograd must see the layer: a training-mode call while grad is recorded and an input
    or weight requires grad."""
    if is_inference_mode_enabled or not torch.is_grad_enabled():
        return False
    return any(isinstance(t, torch.Tensor) and t.requires_grad for t in tensors)


class _FP8MoEFunction(torch.autograd.Function):
    """Training forward + FP8 backward of the token-choice layer after the router GEMM (the reference's
    router function, _UpProjection and _DownProjection autograd functions,
    functional/__init__.py:174-202, 227-479).  Inputs: x [T, H] bf16, router_logits [T, E], w1 / w2 in
    the reference's (2I, H, E) / (H, I, E) views (interleaved or concatenated gate/up rows); outputs
    (o, expert_frequency)."""

    @staticmethod
    def forward(ctx, x, router_logits, w1, w2, K, softmax_over_topk, norm_topk_probs, concat_layout):
        w1q = prepare_fp8_weights(w1, concat_glu=concat_layout, with_t=True)
        w2q = prepare_fp8_weights(w2, concat_glu=False, with_t=True)
        T, H = x.shape
        E = router_logits.shape[1]
        I = w1q.shape[1] // 2
        dev = x.device
        err = torch.zeros(1, dtype=torch.int32, device=dev)
        scores, idx = ops.router_topk(router_logits, K, softmax_over_topk, norm_topk_probs)
        plan = ops.route_plan(idx, E, err)
        xq, xsf = ops.quant_pack(x, idx, plan)
        h = torch.empty(T * K, 2 * I, dtype=torch.bfloat16, device=dev)
        aq, asf = ops.moe_up(xq, xsf, w1q, plan, err, preact_out=h)
        del xq, xsf
        out = torch.zeros(T, H, dtype=torch.bfloat16, device=dev)
        ops.moe_down_combine(aq, asf, w2q, plan, scores, T, err, out=out)
        ctx.save_for_backward(x, router_logits, w1, w2, scores, idx, h, err, plan.freq, plan.off, plan.x_gather,
                              plan.s_scatter, plan.s_rev, plan.off_pad, plan.blk_expert, plan.n_blocks)
        ctx.max_blocks = plan.max_blocks
        ctx.modes = (bool(softmax_over_topk), bool(norm_topk_probs), bool(concat_layout))
        freq = plan.freq.clone()
        ctx.mark_non_differentiable(freq)
        return out, freq

    @staticmethod
    def backward(ctx, dout, _dfreq):
        (x, router_logits, w1, w2, scores, idx, h, err, freq, off, x_gather, s_scatter, s_rev, off_pad, blk_expert,
         n_blocks) = ctx.saved_tensors
        plan = ops.RoutePlan(freq, off, x_gather, s_scatter, s_rev, off_pad, blk_expert, n_blocks, ctx.max_blocks)
        sot, norm, concat = ctx.modes
        # the e4m3 weights the forward ran with (cached per weight version), read transposed
        w1q = prepare_fp8_weights(w1, concat_glu=concat)
        w2q = prepare_fp8_weights(w2, concat_glu=False)
        dx, dlogits, dw1, dw2, _ = ops.moe_backward(dout.to(torch.bfloat16).contiguous(), x, router_logits, w1q, w2q,
                                                    scores, idx, plan, h, sot, norm, err)
        code = int(err.item())
        if code:
            raise RuntimeError(f"FP8 MoE backward: device error {code}")
        return (dx, dlogits.to(router_logits.dtype), dw1.permute(1, 2, 0).to(w1.dtype), dw2.permute(1, 2, 0).to(w2.dtype),
                None, None, None, None)


@torch.library.custom_op("sonicmoe::fp8_moe_tc_forward", mutates_args=())
def _fp8_moe_tc_forward(
    x: torch.Tensor,
    router_logits: torch.Tensor,
    w1: torch.Tensor,
    w2: torch.Tensor,
    K: int,
    is_softmax_over_topk: bool,
    norm_topk_probs: bool,
    concat_layout: bool,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Engine part of ``moe_TC_softmax_topk_layer`` after the router GEMM: (o [T, H] bf16,
    expert_frequency [E] int32).  w1 / w2 are the reference's (2I, H, E) / (H, I, E) views."""
    w1q = prepare_fp8_weights(w1, concat_glu=concat_layout)
    w2q = prepare_fp8_weights(w2, concat_glu=False)
    return ops.moe_forward(x, router_logits, w1q, w2q, K, is_softmax_over_topk, norm_topk_probs)


@_fp8_moe_tc_forward.register_fake
def _(x, router_logits, w1, w2, K, is_softmax_over_topk, norm_topk_probs, concat_layout):
    return x.new_empty(x.shape, dtype=torch.bfloat16), x.new_empty(router_logits.shape[1], dtype=torch.int32)


@torch.library.custom_op("sonicmoe::fp8_moe_tc_forward_fused_router", mutates_args=())
def _fp8_moe_tc_forward_fused_router(
    x: torch.Tensor,
    router_w: torch.Tensor,
    w1: torch.Tensor,
    w2: torch.Tensor,
    K: int,
    is_softmax_over_topk: bool,
    norm_topk_probs: bool,
    concat_layout: bool,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``moe_TC_softmax_topk_layer`` with the fused router (router GEMM + top-k in one kernel):
    (o [T, H] bf16, router_logits [T, E] bf16, expert_frequency [E] int32)."""
    w1q = prepare_fp8_weights(w1, concat_glu=concat_layout)
    w2q = prepare_fp8_weights(w2, concat_glu=False)
    return ops.moe_forward_fused_router(x, router_w, w1q, w2q, K, is_softmax_over_topk, norm_topk_probs)


@_fp8_moe_tc_forward_fused_router.register_fake
def _(x, router_w, w1, w2, K, is_softmax_over_topk, norm_topk_probs, concat_layout):
    E = router_w.shape[0]
    return (x.new_empty(x.shape, dtype=torch.bfloat16), x.new_empty((x.shape[0], E), dtype=torch.bfloat16),
            x.new_empty(E, dtype=torch.int32))


@torch.library.custom_op("sonicmoe::fp8_moe_general_forward", mutates_args=())
def _fp8_moe_general_forward(
    x: torch.Tensor,
    router_scores: torch.Tensor,
    token_indices: torch.Tensor,
    expert_indices: torch.Tensor,
    w1: torch.Tensor,
    w2: torch.Tensor,
    concat_layout: bool,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Engine part of ``moe_general_routing_inputs``: (o [T, H] bf16, expert_frequency [E] int32)."""
    w1q = prepare_fp8_weights(w1, concat_glu=concat_layout)
    w2q = prepare_fp8_weights(w2, concat_glu=False)
    return ops.moe_general_forward(x, router_scores, token_indices, expert_indices, w1q, w2q)


@_fp8_moe_general_forward.register_fake
def _(x, router_scores, token_indices, expert_indices, w1, w2, concat_layout):
    return x.new_empty(x.shape, dtype=torch.bfloat16), x.new_empty(w2.shape[-1], dtype=torch.int32)


def _int4_parts(w1, w2):
    """A pair of prepared 4-bit weights taken apart, as the registered ops below take it."""
    return w1.q, w1.scales, w2.q, w2.scales, list(w1.shape), list(w2.shape), w1.group_size, w2.group_size


def _int4_whole(w1q, w1_scales, w2q, w2_scales, w1_shape, w2_shape, w1_group, w2_group):
    # concat_glu only says how the caller's rows were ordered before they were prepared
    return (Int4ExpertWeights(w1q, w1_scales, tuple(w1_shape), w1_group, False),
            Int4ExpertWeights(w2q, w2_scales, tuple(w2_shape), w2_group, False))


def _int4_tc(x, router_logits, w1, w2, K, is_softmax_over_topk, norm_topk_probs):
    scores, idx = ops.router_topk(router_logits, K, is_softmax_over_topk, norm_topk_probs)
    return ops.moe_int4_forward(x, scores, idx, w1, w2)


def _int4_tc_fused_router(x, router_w, w1, w2, K, is_softmax_over_topk, norm_topk_probs):
    router_logits, scores, idx = ops.router_fused(x, router_w, K, is_softmax_over_topk, norm_topk_probs)
    o, expert_frequency = ops.moe_int4_forward(x, scores, idx, w1, w2)
    return o, router_logits, expert_frequency


@torch.library.custom_op("sonicmoe::int4_moe_tc_forward", mutates_args=())
def _int4_moe_tc_forward(
    x: torch.Tensor,
    router_logits: torch.Tensor,
    w1q: torch.Tensor,
    w1_scales: torch.Tensor,
    w2q: torch.Tensor,
    w2_scales: torch.Tensor,
    w1_shape: list[int],
    w2_shape: list[int],
    w1_group: int,
    w2_group: int,
    K: int,
    is_softmax_over_topk: bool,
    norm_topk_probs: bool,
) -> tuple[torch.Tensor, torch.Tensor]:
    """``moe_TC_softmax_topk_layer`` after the router GEMM on 4-bit expert weights (the prepared
    ``Int4ExpertWeights`` taken apart): (o [T, H] bf16, expert_frequency [E] int32)."""
    w1, w2 = _int4_whole(w1q, w1_scales, w2q, w2_scales, w1_shape, w2_shape, w1_group, w2_group)
    return _int4_tc(x, router_logits, w1, w2, K, is_softmax_over_topk, norm_topk_probs)


@_int4_moe_tc_forward.register_fake
def _(x, router_logits, w1q, w1_scales, w2q, w2_scales, w1_shape, w2_shape, w1_group, w2_group, K,
      is_softmax_over_topk, norm_topk_probs):
    return x.new_empty(x.shape, dtype=torch.bfloat16), x.new_empty(router_logits.shape[1], dtype=torch.int32)


@torch.library.custom_op("sonicmoe::int4_module_forward", mutates_args=())
def _int4_module_forward(
    x: torch.Tensor,
    router_logits: torch.Tensor,
    w1: torch.Tensor,
    w2: torch.Tensor,
    handle: int,
    K: int,
) -> tuple[torch.Tensor, torch.Tensor]:
    """The layer after the router GEMM on the ``Int4Copies`` of that number, of the module's weights w1 [E, 2I, H]
    and w2 [E, H, I] as they are when the graph runs."""
    return _int4_tc(x, router_logits, *Int4Copies._known[handle].current(w1, w2), K, True, False)


@_int4_module_forward.register_fake
def _(x, router_logits, w1, w2, handle, K):
    return x.new_empty(x.shape, dtype=torch.bfloat16), x.new_empty(router_logits.shape[1], dtype=torch.int32)


@torch.library.custom_op("sonicmoe::int4_moe_tc_forward_fused_router", mutates_args=())
def _int4_moe_tc_forward_fused_router(
    x: torch.Tensor,
    router_w: torch.Tensor,
    w1q: torch.Tensor,
    w1_scales: torch.Tensor,
    w2q: torch.Tensor,
    w2_scales: torch.Tensor,
    w1_shape: list[int],
    w2_shape: list[int],
    w1_group: int,
    w2_group: int,
    K: int,
    is_softmax_over_topk: bool,
    norm_topk_probs: bool,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The same with the fused router: (o [T, H] bf16, router_logits [T, E] bf16, expert_frequency [E] int32)."""
    w1, w2 = _int4_whole(w1q, w1_scales, w2q, w2_scales, w1_shape, w2_shape, w1_group, w2_group)
    return _int4_tc_fused_router(x, router_w, w1, w2, K, is_softmax_over_topk, norm_topk_probs)


@_int4_moe_tc_forward_fused_router.register_fake
def _(x, router_w, w1q, w1_scales, w2q, w2_scales, w1_shape, w2_shape, w1_group, w2_group, K,
      is_softmax_over_topk, norm_topk_probs):
    E = router_w.shape[0]
    return (x.new_empty(x.shape, dtype=torch.bfloat16), x.new_empty((x.shape[0], E), dtype=torch.bfloat16),
            x.new_empty(E, dtype=torch.int32))


@torch.library.custom_op("sonicmoe::int4_moe_general_forward", mutates_args=())
def _int4_moe_general_forward(
    x: torch.Tensor,
    router_scores: torch.Tensor,
    token_indices: torch.Tensor,
    expert_indices: torch.Tensor,
    w1q: torch.Tensor,
    w1_scales: torch.Tensor,
    w2q: torch.Tensor,
    w2_scales: torch.Tensor,
    w1_shape: list[int],
    w2_shape: list[int],
    w1_group: int,
    w2_group: int,
) -> tuple[torch.Tensor, torch.Tensor]:
    """``moe_general_routing_inputs`` on 4-bit expert weights: (o [T, H] bf16, expert_frequency [E] int32)."""
    w1, w2 = _int4_whole(w1q, w1_scales, w2q, w2_scales, w1_shape, w2_shape, w1_group, w2_group)
    return ops.moe_int4_general_forward(x, router_scores, token_indices, expert_indices, w1, w2)


@_int4_moe_general_forward.register_fake
def _(x, router_scores, token_indices, expert_indices, w1q, w1_scales, w2q, w2_scales, w1_shape, w2_shape, w1_group,
      w2_group):
    return x.new_empty(x.shape, dtype=torch.bfloat16), x.new_empty(w2_shape[0], dtype=torch.int32)


class _FP8MoEGeneralFunction(torch.autograd.Function):
    """Training forward + FP8 backward of the layer over explicit routing lists
    (``moe_general_routing_inputs``, reference functional/__init__.py:571-652 with its autograd
    functions): gradients for x, the router scores and the expert weights."""

    @staticmethod
    def forward(ctx, x, router_scores, token_indices, expert_indices, w1, w2, concat_layout):
        w1q = prepare_fp8_weights(w1, concat_glu=concat_layout, with_t=True)
        w2q = prepare_fp8_weights(w2, concat_glu=False, with_t=True)
        T, H = x.shape
        E = w2q.shape[0]
        I = w2q.shape[2]
        TK = router_scores.numel()
        dev = x.device
        err = torch.zeros(1, dtype=torch.int32, device=dev)
        plan = ops.general_route_plan(token_indices, expert_indices, T, E, err)
        xq, xsf = ops.quant_pack_general(x, expert_indices, plan)
        h = torch.empty(TK, 2 * I, dtype=torch.bfloat16, device=dev)
        aq, asf = ops.moe_up(xq, xsf, w1q, plan, err, preact_out=h)
        del xq, xsf
        out = torch.zeros(T, H, dtype=torch.bfloat16, device=dev)
        ops.moe_down_combine(aq, asf, w2q, plan, router_scores, T, err, out=out)
        ctx.save_for_backward(x, router_scores, expert_indices, w1, w2, h, err, plan.freq, plan.off, plan.x_gather,
                              plan.s_scatter, plan.s_rev, plan.off_pad, plan.blk_expert, plan.n_blocks, plan.tok_off)
        ctx.max_blocks = plan.max_blocks
        ctx.concat = bool(concat_layout)
        freq = plan.freq.clone()
        ctx.mark_non_differentiable(freq)
        return out, freq

    @staticmethod
    def backward(ctx, dout, _dfreq):
        (x, router_scores, expert_indices, w1, w2, h, err, freq, off, x_gather, s_scatter, s_rev, off_pad,
         blk_expert, n_blocks, tok_off) = ctx.saved_tensors
        plan = ops.RoutePlan(freq, off, x_gather, s_scatter, s_rev, off_pad, blk_expert, n_blocks, ctx.max_blocks,
                             tok_off)
        w1q = prepare_fp8_weights(w1, concat_glu=ctx.concat)
        w2q = prepare_fp8_weights(w2, concat_glu=False)
        dx, _, dw1, dw2, ds = ops.moe_backward(dout.to(torch.bfloat16).contiguous(), x, None, w1q, w2q,
                                               router_scores, expert_indices, plan, h, True, False, err, general=True)
        code = int(err.item())
        if code:
            raise RuntimeError(f"FP8 MoE backward: device error {code}")
        return (dx, ds.to(router_scores.dtype), None, None, dw1.permute(1, 2, 0).to(w1.dtype),
                dw2.permute(1, 2, 0).to(w2.dtype), None)


def moe_TC_softmax_topk_layer(
    x: torch.Tensor,
    router_w: torch.Tensor,
    w1,
    b1,
    w2,
    b2,
    K: int,
    stream_id: int,
    activation_type=ActivationType.SWIGLU,
    is_inference_mode_enabled: bool = False,
    is_softmax_over_topk: bool = True,
    norm_topk_probs: bool = False,
    concat_layout: bool = False,
    *,
    fused_router: bool = False,
):
    """Token-choice top-k MoE layer forward.  Returns (o [T, H], router_logits [T, E], expert_frequency [E]).

    ``stream_id`` is ignored, as in the reference (the current torch stream is used).

    ``fused_router`` (keyword only; not in the reference): compute the router logits and their top-k
    in one tcgen05 kernel instead of ``F.linear`` + the top-k kernel.  Its logits come from the
    tensor core's fp32 accumulation, so they can differ from ``F.linear``'s in the last bf16 bit (and
    a near-tie can then route to another expert); needs E % 32 == 0, 32 <= E <= 256, H % 64 == 0.
    """
    _check_common(b1, b2, activation_type)
    if norm_topk_probs and is_softmax_over_topk:
        raise ValueError("`norm_topk_prob` only works with softmax-then-topk")
    training = _wants_training(is_inference_mode_enabled, x, router_w, w1, w2)
    if training and (fused_router or _prepared(w1) or _prepared(w2)):
        raise NotImplementedError("the FP8 backward covers bf16 weights with the F.linear router "
                                  "(no fused_router or prepared weights)")
    int4 = _int4_pair(w1, w2, concat_layout)
    if x.dtype != torch.bfloat16:
        x = x.to(torch.bfloat16)
    x = x.contiguous()
    if int4:
        traced = torch.compiler.is_compiling()
        modes = (K, is_softmax_over_topk, norm_topk_probs)
        if fused_router:
            rw = router_w.to(x.dtype).contiguous()
            if traced:
                return _int4_moe_tc_forward_fused_router(x, rw, *_int4_parts(w1, w2), *modes)
            return _int4_tc_fused_router(x, rw, w1, w2, *modes)
        router_logits = F.linear(x, router_w.to(x.dtype))
        if traced:
            o, expert_frequency = _int4_moe_tc_forward(x, router_logits.contiguous(), *_int4_parts(w1, w2), *modes)
        else:
            o, expert_frequency = _int4_tc(x, router_logits.contiguous(), w1, w2, *modes)
        return o, router_logits, expert_frequency
    if training:
        router_logits = F.linear(x, router_w.to(x.dtype))
        o, expert_frequency = _FP8MoEFunction.apply(x, router_logits, w1, w2, K, is_softmax_over_topk,
                                                    norm_topk_probs, concat_layout)
        return o, router_logits, expert_frequency
    if fused_router:
        rw = router_w.to(x.dtype).contiguous()
        if isinstance(w1, Fp8ExpertWeights) or isinstance(w2, Fp8ExpertWeights):
            w1q = prepare_fp8_weights(w1, concat_glu=concat_layout)
            w2q = prepare_fp8_weights(w2, concat_glu=False)
            if w1q.concat_glu != bool(concat_layout):
                raise ValueError("prepared w1 layout does not match concat_layout")
            o, router_logits, expert_frequency = ops.moe_forward_fused_router(
                x, rw, w1q, w2q, K, is_softmax_over_topk, norm_topk_probs)
        else:
            o, router_logits, expert_frequency = _fp8_moe_tc_forward_fused_router(
                x, rw, w1, w2, K, is_softmax_over_topk, norm_topk_probs, concat_layout)
        return o, router_logits, expert_frequency
    router_logits = F.linear(x, router_w.to(x.dtype))
    if isinstance(w1, Fp8ExpertWeights) or isinstance(w2, Fp8ExpertWeights):
        # already prepared e4m3 weights (a host-side object, not a tensor): eager call
        w1q = prepare_fp8_weights(w1, concat_glu=concat_layout)
        w2q = prepare_fp8_weights(w2, concat_glu=False)
        if w1q.concat_glu != bool(concat_layout):
            raise ValueError("prepared w1 layout does not match concat_layout")
        o, expert_frequency = ops.moe_forward(
            x, router_logits.contiguous(), w1q, w2q, K, is_softmax_over_topk, norm_topk_probs
        )
    else:
        o, expert_frequency = _fp8_moe_tc_forward(
            x, router_logits.contiguous(), w1, w2, K, is_softmax_over_topk, norm_topk_probs, concat_layout
        )
    return o, router_logits, expert_frequency


def int4_module_layer(x, router_w, w1, b1, w2, b2, K: int, copies: Int4Copies, activation_type=ActivationType.SWIGLU,
                      is_inference_mode_enabled: bool = False):
    """``moe_TC_softmax_topk_layer`` on the 4-bit copies of a module's weights w1 [E, 2I, H] and w2 [E, H, I], brought
    up to date."""
    if not torch.compiler.is_compiling() or copies.away(w1, w2):
        q1, q2 = copies.copies if torch.compiler.is_compiling() else copies.current(w1, w2)
        return moe_TC_softmax_topk_layer(x, router_w, q1, b1, q2, b2, K, None, activation_type, is_inference_mode_enabled)
    _check_common(b1, b2, activation_type)
    if _wants_training(is_inference_mode_enabled, x, router_w):
        raise NotImplementedError("4-bit expert weights have no backward")
    x = x.to(torch.bfloat16).contiguous()
    router_logits = F.linear(x, router_w.to(x.dtype))
    o, expert_frequency = _int4_module_forward(x, router_logits.contiguous(), w1.detach(), w2.detach(), copies.handle, K)
    return o, router_logits, expert_frequency


def moe_general_routing_inputs(
    x: torch.Tensor,
    router_scores: torch.Tensor,
    token_indices: torch.Tensor,
    expert_indices: torch.Tensor,
    w1,
    b1,
    w2,
    b2,
    E: int,
    stream_id: int,
    activation_type=ActivationType.SWIGLU,
    is_inference_mode_enabled: bool = False,
    concat_layout: bool = False,
):
    """MoE forward from explicit (token, expert, score) lists; token_indices must be sorted ascending.

    Returns (o [T, H], expert_frequency [E]).  ``E`` is taken from ``w2`` as in the reference
    (``functional/__init__.py:592``).
    """
    _check_common(b1, b2, activation_type)
    training = _wants_training(is_inference_mode_enabled, x, router_scores, w1, w2)
    if training and (_prepared(w1) or _prepared(w2)):
        raise NotImplementedError("the FP8 backward covers bf16 weights (no prepared weights)")
    int4 = _int4_pair(w1, w2, concat_layout)
    if x.dtype != torch.bfloat16:
        x = x.to(torch.bfloat16)
    x = x.contiguous()
    if router_scores.dtype != torch.float32:
        router_scores = router_scores.float()
    args = (x, router_scores.contiguous(), token_indices.to(torch.int32).contiguous(),
            expert_indices.to(torch.int32).contiguous())
    if int4:
        if torch.compiler.is_compiling():
            return _int4_moe_general_forward(*args, *_int4_parts(w1, w2))
        return ops.moe_int4_general_forward(*args, w1, w2)
    if training:
        return _FP8MoEGeneralFunction.apply(*args, w1, w2, concat_layout)
    if isinstance(w1, Fp8ExpertWeights) or isinstance(w2, Fp8ExpertWeights):
        w1q = prepare_fp8_weights(w1, concat_glu=concat_layout)
        w2q = prepare_fp8_weights(w2, concat_glu=False)
        return ops.moe_general_forward(*args, w1q, w2q)
    return _fp8_moe_general_forward(*args, w1, w2, concat_layout)


def _has_tangent(t) -> bool:
    return fwAD._current_level >= 0 and fwAD.unpack_dual(t).tangent is not None


def _switch_loss_gradient(router_logits, coef, token_mask):
    """dloss/dlogits [T, E] fp32 in torch operations, which any transform can follow."""
    z, on = router_logits, None
    if token_mask is not None:  # what a left-out row holds must not reach a second gradient either
        on = token_mask[:, None] != 0
        z = z.where(on, 0.0)
    p = F.softmax(z, dim=-1, dtype=torch.float32)
    if on is not None:
        p = p.where(on, 0.0)
    return p * (coef - (p * coef).sum(-1, keepdim=True))


class _SwitchLossFunction(torch.autograd.Function):
    """Balance loss with its derivatives for the router logits; the counts carry none."""

    @staticmethod
    def forward(ctx, router_logits, expert_frequency, topk_indices, token_mask):
        loss, freq, coef = ops.switch_loss(router_logits, expert_frequency, topk_indices, token_mask)
        ctx.save_for_backward(router_logits, coef, token_mask)
        ctx.save_for_forward(router_logits, coef, token_mask)
        ctx.mark_non_differentiable(freq)
        ctx.set_materialize_grads(False)
        return loss, freq

    @staticmethod
    def backward(ctx, dloss, *_):
        if dloss is None:
            return None, None, None, None
        router_logits, coef, token_mask = ctx.saved_tensors
        # create_graph, a transform around this, a batch of gradients (which has no storage to point to) or forward
        # mode through the backward: the same formula in operations that can be followed
        if (torch.is_grad_enabled() or torch._C._are_functorch_transforms_active()
                or torch._C._functorch.is_legacy_batchedtensor(dloss) or _has_tangent(router_logits)
                or _has_tangent(dloss)):
            dl = dloss * _switch_loss_gradient(router_logits, coef, token_mask)
            return dl.to(router_logits.dtype), None, None, None
        return ops.switch_loss_bwd(router_logits, coef, dloss.to(torch.float32), token_mask), None, None, None

    @staticmethod
    def jvp(ctx, tangent, counts_tangent, *_):
        if counts_tangent is not None:
            raise NotImplementedError("expert_frequency carries no derivative; give it without a tangent")
        if tangent is None:
            return None, None
        return (_switch_loss_gradient(*ctx.saved_tensors) * tangent).sum(), None


class _SwitchLossTransformed(_SwitchLossFunction):
    """The same for torch.func's transforms, which need the context set up apart and a rule for batches.  (Apart,
    since such a function costs an eager call 30 us more.)"""

    @staticmethod
    def forward(router_logits, expert_frequency, topk_indices, token_mask):
        return ops.switch_loss(router_logits, expert_frequency, topk_indices, token_mask)

    @staticmethod
    def setup_context(ctx, inputs, output):
        router_logits, _, _, token_mask = inputs
        _, freq, coef = output
        ctx.save_for_backward(router_logits, coef, token_mask)
        ctx.save_for_forward(router_logits, coef, token_mask)
        ctx.mark_non_differentiable(freq, coef)
        ctx.set_materialize_grads(False)

    @staticmethod
    def jvp(ctx, *tangents):
        return *_SwitchLossFunction.jvp(ctx, *tangents), None

    @staticmethod
    def vmap(info, in_dims, *args):
        outs = [_SwitchLossTransformed.apply(*(a if d is None else a.select(d, i).contiguous()
                                               for a, d in zip(args, in_dims))) for i in range(info.batch_size)]
        return tuple(torch.stack(o) for o in zip(*outs)), (0, 0, 0)


@torch.library.custom_op("sonicmoe::switch_loss", mutates_args=())
def _switch_loss_op(
    router_logits: torch.Tensor,
    expert_frequency: torch.Tensor | None,
    topk_indices: torch.Tensor | None,
    token_mask: torch.Tensor | None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``ops.switch_loss`` for traced callers: (loss fp32 [], counts [E], coef fp32 [E])."""
    return ops.switch_loss(router_logits, expert_frequency, topk_indices, token_mask)


@_switch_loss_op.register_fake
def _(router_logits, expert_frequency, topk_indices, token_mask):
    E = router_logits.shape[1]
    counts = torch.int32 if expert_frequency is None else expert_frequency.dtype
    return (router_logits.new_empty((), dtype=torch.float32), router_logits.new_empty(E, dtype=counts),
            router_logits.new_empty(E, dtype=torch.float32))


@torch.library.custom_op("sonicmoe::switch_loss_bwd", mutates_args=())
def _switch_loss_bwd_op(router_logits: torch.Tensor, coef: torch.Tensor, dloss: torch.Tensor,
                        token_mask: torch.Tensor | None) -> torch.Tensor:
    return ops.switch_loss_bwd(router_logits, coef, dloss, token_mask)


@_switch_loss_bwd_op.register_fake
def _(router_logits, coef, dloss, token_mask):
    return torch.empty_like(router_logits)


def _switch_loss_setup(ctx, inputs, output):
    ctx.save_for_backward(inputs[0], output[2], inputs[3])


def _switch_loss_backward(ctx, dloss, _dfreq, _dcoef):
    router_logits, coef, token_mask = ctx.saved_tensors
    return _switch_loss_bwd_op(router_logits, coef, dloss.to(torch.float32), token_mask), None, None, None


_switch_loss_op.register_autograd(_switch_loss_backward, setup_context=_switch_loss_setup)


# exact conversions of given counts to a type the kernels read
_COUNT_AS = {torch.bool: torch.int32, torch.uint8: torch.int32, torch.int8: torch.int32, torch.int16: torch.int32,
             torch.float16: torch.float32, torch.bfloat16: torch.float32}


def _given_counts(expert_frequency):
    if expert_frequency.dtype is torch.int32:
        return expert_frequency.contiguous()
    if expert_frequency.is_floating_point():
        if expert_frequency.requires_grad and torch.is_grad_enabled() or _has_tangent(expert_frequency):
            raise ValueError("expert_frequency gets no gradient; give it detached")
    dtype = _COUNT_AS.get(expert_frequency.dtype, expert_frequency.dtype)
    if dtype not in ops._COUNT_TYPES:
        raise ValueError(f"expert_frequency must hold whole or real numbers, got {expert_frequency.dtype}")
    return expert_frequency.to(dtype).contiguous()


def _expert_ids(topk_indices, E):
    if topk_indices.is_floating_point() or topk_indices.is_complex():
        raise ValueError(f"topk_indices must hold whole numbers, got {topk_indices.dtype}")
    if topk_indices.dtype == torch.int64:  # an id that int32 cannot hold must not become a valid one
        topk_indices = topk_indices.clamp(-1, E)
    return topk_indices.to(torch.int32).contiguous()


def switch_load_balancing_loss(
    router_logits: torch.Tensor,
    expert_frequency: torch.Tensor | None = None,
    topk_indices: torch.Tensor | None = None,
    token_mask: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Switch load-balancing loss of the router (the formula of reference moe.py:263-276) and the experts'
    counts: (loss fp32 [], expert_frequency [E]), differentiable with respect to router_logits (backward,
    forward mode, torch.func's transforms, and any of them again).

        p = softmax(router_logits), loss = E * sum_e (sum_t p[t, e] / sum p) (f_e / sum f)

    Args:
        router_logits: [T, E], bf16, fp16 or fp32.
        expert_frequency: [E] counts f, as ``moe_TC_softmax_topk_layer`` returns them, or any numbers >= 0
            in their proportions (fractions of the entries, counts averaged over ranks); or
        topk_indices: [T, K] expert ids, as ``ops.router_topk`` returns them, which are counted here in int32.
            Exactly one of the two is given; neither gets a gradient.
        token_mask: [T] bool, optional: tokens that are False (padding) take no part in the
            probabilities, in the counts made from topk_indices, or in the gradient.

    The loss is 0 when no token or no entry counts.  The same inputs give the same bits.
    """
    router_logits = router_logits.contiguous()
    if expert_frequency is not None:
        expert_frequency = _given_counts(expert_frequency)
    if topk_indices is not None:
        topk_indices = _expert_ids(topk_indices, router_logits.shape[-1])
    if token_mask is not None:
        token_mask = token_mask.contiguous()
    if torch.compiler.is_compiling():
        loss, freq, _ = _switch_loss_op(router_logits, expert_frequency, topk_indices, token_mask)
    elif torch._C._are_functorch_transforms_active():
        loss, freq, _ = _SwitchLossTransformed.apply(router_logits, expert_frequency, topk_indices, token_mask)
    elif router_logits.requires_grad and torch.is_grad_enabled() or _has_tangent(router_logits):
        loss, freq = _SwitchLossFunction.apply(router_logits, expert_frequency, topk_indices, token_mask)
    else:
        loss, freq, _ = ops.switch_loss(router_logits, expert_frequency, topk_indices, token_mask)
    return loss, freq


@torch.library.custom_op(
    "triton_kernels::TC_topk_router_metadata",
    mutates_args={"expert_frequency", "expert_frequency_offset", "x_gather_idx", "s_scatter_idx",
                  "s_reverse_scatter_idx"},
)
def TC_topk_router_metadata_triton(
    topk_router_indices: torch.Tensor,
    E: int,
    expert_frequency: torch.Tensor,
    expert_frequency_offset: torch.Tensor,
    x_gather_idx: torch.Tensor,
    s_scatter_idx: torch.Tensor,
    s_reverse_scatter_idx: torch.Tensor,
) -> None:
    """Reference op and signature (triton_kernels/__init__.py:68-86): fills the five int32 outputs in
    place (directly when they are contiguous int32, else through a copy)."""
    outs = (expert_frequency, expert_frequency_offset, x_gather_idx, s_scatter_idx, s_reverse_scatter_idx)
    idx = topk_router_indices.to(torch.int32).contiguous()
    if all(t.dtype == torch.int32 and t.is_contiguous() for t in outs):
        ops.route_metadata(idx, E, outs=outs)
        return
    for dst, src in zip(outs, ops.route_metadata(idx, E)):
        dst.copy_(src)


@torch.library.custom_op(
    "triton_kernels::general_routing_router_metadata",
    mutates_args={"expert_frequency", "expert_frequency_offset", "x_gather_idx", "s_scatter_idx",
                  "s_reverse_scatter_idx", "num_activated_expert_per_token_offset"},
)
def general_routing_router_metadata_triton(
    sorted_selected_T: torch.Tensor,
    selected_E: torch.Tensor,
    T: int,
    E: int,
    expert_frequency: torch.Tensor,
    expert_frequency_offset: torch.Tensor,
    x_gather_idx: torch.Tensor,
    s_scatter_idx: torch.Tensor,
    s_reverse_scatter_idx: torch.Tensor,
    num_activated_expert_per_token_offset: torch.Tensor,
) -> None:
    """Reference op and signature (triton_kernels/__init__.py:270-292): fills the six int32 outputs in place."""
    outs = (expert_frequency, expert_frequency_offset, x_gather_idx, s_scatter_idx, s_reverse_scatter_idx,
            num_activated_expert_per_token_offset)
    tok = sorted_selected_T.to(torch.int32).contiguous()
    ex = selected_E.to(torch.int32).contiguous()
    if all(t.dtype == torch.int32 and t.is_contiguous() for t in outs):
        ops.general_route_metadata(tok, ex, T, E, outs=outs)
        return
    for dst, src in zip(outs, ops.general_route_metadata(tok, ex, T, E)):
        dst.copy_(src)
