"""Declared support surface of the operator and the one exception a caller may catch.

Mirror of the reference's src/attn_kernel_lab/capability.py:21-253 -- same class names,
fields, check order and message shape -- so code written against the reference's surface
runs unchanged.  `CapabilityError` (a `ValueError`) means "this request is outside the
declared surface, route it elsewhere"; any other exception is a defect.
"""
from __future__ import annotations

from dataclasses import dataclass, field


class CapabilityError(ValueError):
    """The request is outside the declared surface (capability.py:21-33 of the reference)."""

    def __init__(self, message: str, *, field: str, value: object, supported: object):
        super().__init__(message)
        self.field = field
        self.value = value
        self.supported = supported


@dataclass(frozen=True)
class OperatorCapability:
    """What one contract version accepts (capability.py:36-52)."""

    operator_contract_version: int
    layout_version: int
    head_dim: tuple[int, ...]
    q_heads: tuple[int, ...]
    kv_heads: tuple[int, ...]
    page_size: tuple[int, ...]
    modes: tuple[str, ...]
    masks: tuple[str, ...]
    returns_lse: bool = False
    kv_dtypes: tuple[str, ...] = ("bfloat16", "float16")
    cuda_graph: str = "supported"
    notes: tuple[str, ...] = field(default_factory=tuple)


#: GQA pairs with numerical test coverage; the declared family is the kv_heads = 4 part of it,
#: because the schema is per axis and would otherwise admit untested cross pairs
#: (capability.py:88-113).
TESTED_GQA_RATIOS = ((8, 2), (16, 4), (24, 4), (32, 4))
DECLARED_GQA_RATIOS = ((16, 4), (24, 4), (32, 4))
CUDA_GRAPH_DECLARED = "supported"

#: Workspace byte layout of this implementation: 128-byte-swizzled tensor-core tile images
#: (Q8/K8 as [tile][2][128][128], V8 transposed as [pair][256][128]).  The reference's layout 1
#: (SIGMA64-permuted mma.sync fragments, quant.py:95-100) is not part of the operator
#: (docs/OPERATOR_CONTRACT.md:151-167), so this is a new layout version, not a new contract.
LAYOUT_VERSION = 2


def _axes(pairs):
    return (tuple(sorted({q for q, _ in pairs})), tuple(sorted({kv for _, kv in pairs})))


_V1_Q, _V1_KV = _axes(DECLARED_GQA_RATIOS)
_GEN_Q, _GEN_KV = _axes(TESTED_GQA_RATIOS)

V1_CAPABILITY = OperatorCapability(
    operator_contract_version=1,
    layout_version=LAYOUT_VERSION,
    head_dim=(256,),
    q_heads=_V1_Q,
    kv_heads=_V1_KV,
    page_size=(1,),
    modes=("extend",),
    masks=("bottom_right_causal",),
    returns_lse=True,
    kv_dtypes=("bfloat16", "float16"),
    cuda_graph=CUDA_GRAPH_DECLARED,
    notes=(
        "E4M3 V and P on sm_100a; Q and K in INT8 (qk_i8=True, the default, as in the reference) or "
        "E4M3 (qk_i8=False, the mode the throughput figures are quoted in).",
        "CUDA graph capture needs a capacity-reserved workspace (plan_workspace) and "
        "caller-owned out / lse_out.",
        "An FP8 or FP4 KV pool would be quantised twice and is refused.",
    ),
)

#: Test-only widening of the head axes (capability.py:187-215); never a production surface.
GENERALIZATION_CAPABILITY = OperatorCapability(
    operator_contract_version=1,
    layout_version=LAYOUT_VERSION,
    head_dim=(256,),
    q_heads=tuple(sorted(set(_GEN_Q))),
    kv_heads=tuple(sorted(set(_GEN_KV) | {1})),
    page_size=(1,),
    modes=("extend",),
    masks=("bottom_right_causal",),
    returns_lse=False,
    kv_dtypes=("bfloat16", "float16"),
    cuda_graph=CUDA_GRAPH_DECLARED,
    notes=("Generalisation sweep only: widens q_heads / kv_heads so GQA ratios outside the "
           "declared family can be exercised through the public entry point.",),
)


#: What one KV-head-group shard of a declared request looks like: the q heads of 1 or 2 of the 4 kv
#: heads.  Query heads [j*g, (j+1)*g) read kv head j only and every statistic of the operator is per kv
#: head (docs/OPERATOR_CONTRACT.md:41-42 of the reference; quant.py:516-520), so a request of the
#: declared family splits into such shards with no exchange, each shard's rows bit-identical to the
#: unsharded result.  A caller passes this capability explicitly for the shard calls
#: (`dist.prefill_extend_kv_head_shard` does); the production surface stays V1_CAPABILITY.
KV_HEAD_SHARD_CAPABILITY = OperatorCapability(
    operator_contract_version=1,
    layout_version=LAYOUT_VERSION,
    head_dim=(256,),
    q_heads=tuple(sorted({q // kv * n for q, kv in DECLARED_GQA_RATIOS for n in (1, 2)})),
    kv_heads=(1, 2),
    page_size=(1,),
    modes=("extend",),
    masks=("bottom_right_causal",),
    returns_lse=True,
    kv_dtypes=("bfloat16", "float16"),
    cuda_graph=CUDA_GRAPH_DECLARED,
    notes=("One KV-head-group shard (1 or 2 of the 4 kv heads with their query heads) of a request of the "
           "declared family; results equal the corresponding heads of the unsharded call bit for bit.",),
)


#: Heads of the decode side (`paged_decode`) and of the attention weights of an extend
#: (`extend_weights`): up to eight query heads share a kv head, which covers the declared family, its
#: kv-head shards and the tested ratios.  No counterpart in the reference.
_GROUPS, _DECODE_KV = range(1, 9), (1, 2, 4, 8)
DECODE_CAPABILITY = OperatorCapability(
    operator_contract_version=1,
    layout_version=LAYOUT_VERSION,
    head_dim=(256,),
    q_heads=tuple(sorted({kv * g for kv in _DECODE_KV for g in _GROUPS})),
    kv_heads=_DECODE_KV,
    page_size=(1,),
    modes=("decode", "extend_weights"),
    masks=("bottom_right_causal",),
    returns_lse=True,
    kv_dtypes=("bfloat16", "float16"),
    cuda_graph=CUDA_GRAPH_DECLARED,
    notes=("The pool is read in its own type; nothing is quantised.",
           "CUDA graph capture needs a planned workspace and caller-owned outputs; lengths, rows and "
           "page-table entries are read on the device at replay."),
)


def check_supported(
    *,
    head_dim: int,
    q_heads: int,
    kv_heads: int,
    page_size: int,
    mode: str,
    mask: str,
    kv_dtype: str,
    return_lse: bool = False,
    capability: OperatorCapability = V1_CAPABILITY,
) -> None:
    """Raise `CapabilityError` when a request is outside `capability`.

    Order (capability.py:218-253): head_dim, q_heads, kv_heads, page_size, mode, mask,
    kv_dtype, then LSE, then divisibility."""
    version = capability.operator_contract_version
    for name, value, allowed in (
        ("head_dim", head_dim, capability.head_dim),
        ("q_heads", q_heads, capability.q_heads),
        ("kv_heads", kv_heads, capability.kv_heads),
        ("page_size", page_size, capability.page_size),
        ("mode", mode, capability.modes),
        ("mask", mask, capability.masks),
        ("kv_dtype", kv_dtype, capability.kv_dtypes),
    ):
        if value not in allowed:
            raise CapabilityError(
                f"{name}={value!r} is outside the declared support surface "
                f"{list(allowed)!r} of operator contract v{version}",
                field=name, value=value, supported=allowed,
            )
    if return_lse and not capability.returns_lse:
        raise CapabilityError(
            f"LSE output is not part of operator contract v{version}; an LSE-producing "
            "variant is a new package_api_version, not a flag",
            field="return_lse", value=return_lse, supported=(False,),
        )
    if q_heads % kv_heads:
        raise CapabilityError(
            f"q_heads={q_heads} is not divisible by kv_heads={kv_heads}",
            field="q_heads", value=q_heads, supported=capability.q_heads,
        )
