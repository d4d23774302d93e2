"""The state arena on the GPU: wkvm's RWKV7StateBank with slot-indexed
kernels in place of gather/scatter copies.

Mirrors wkvm/runner/state.py:23-100 and wkvm/models/rwkv7.py:42-99:
  wkv   [L, S+1, H, K, V] fp32   (slot 0 = reserved padding row)
  shift [L, 2, S+1, D] model dtype ([:, 0] attn token-shift, [:, 1] ffn)
Tensors, dtypes and slot semantics are identical, so wkvm's StateStore files
and fingerprints stay compatible. The differences are in how state moves:
decode/prefill kernels read and write ``wkv[layer, slot]`` in place, and
zero / fork / snapshot / restore / migrate are single kernels over all
layers instead of per-layer strided copies.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Mapping, Sequence

import torch

from . import ops, ssm

WKV_DTYPE = torch.float32


@dataclass(frozen=True)
class RWKV7StateLayout:
    """Per-slot state shapes (wkvm/models/rwkv7.py:42-99)."""

    n_layer: int
    hidden_size: int
    num_heads: int
    head_dim: int
    head_v_dim: int
    dtype: torch.dtype = torch.bfloat16

    @property
    def wkv_shape(self) -> tuple[int, ...]:
        return (self.num_heads, self.head_dim, self.head_v_dim)

    @property
    def shift_shape(self) -> tuple[int, ...]:
        return (self.hidden_size,)

    def wkv_bytes_per_slot(self) -> int:
        return self.n_layer * self.num_heads * self.head_dim * self.head_v_dim * 4

    def shift_bytes_per_slot(self) -> int:
        return self.n_layer * 2 * self.hidden_size * torch.empty((), dtype=self.dtype).element_size()


SlotDict = Mapping[str, int]


def _ids(slot_batch: Sequence[SlotDict], family: str) -> list[int]:
    return [int(s[family]) for s in slot_batch]


class RWKV7StateBank:
    """Dense slot-indexed state tensors (wkvm/runner/state.py:23-48)."""

    def __init__(self, layout: RWKV7StateLayout, num_slots: int,
                 device: torch.device | str = "cuda") -> None:
        self.layout = layout
        self.num_slots = num_slots
        self.device = torch.device(device)
        self.wkv = torch.zeros((layout.n_layer, num_slots + 1, *layout.wkv_shape),
                               dtype=WKV_DTYPE, device=self.device)
        self.shift = torch.zeros((layout.n_layer, 2, num_slots + 1, *layout.shift_shape),
                                 dtype=layout.dtype, device=self.device)

    # -- slot lifecycle ---------------------------------------------------

    def zero_slots(self, slots: SlotDict) -> None:
        """wkvm RWKV7StateBank.zero_slots (state.py:50-54): one kernel per family."""
        ops.slot_zero(self.wkv, 1, [int(slots["wkv"])])
        ops.slot_zero(self.shift, 2, [int(slots["shift"])])

    def zero_many(self, slot_batch: Sequence[SlotDict]) -> None:
        ops.slot_zero(self.wkv, 1, _ids(slot_batch, "wkv"))
        ops.slot_zero(self.shift, 2, _ids(slot_batch, "shift"))

    def fork(self, parents: Sequence[SlotDict], children: Sequence[SlotDict]) -> None:
        """Device copy child <- parent for every family (the O(MB) copy wkvm's
        StateArena.fork leaves to the runner, wkvm/core/arena.py:82-92)."""
        ops.slot_copy(self.wkv, 1, _ids(parents, "wkv"), _ids(children, "wkv"))
        ops.slot_copy(self.shift, 2, _ids(parents, "shift"), _ids(children, "shift"))

    # -- mutation rules (wkvm/store.py:260-268, 298-305) on live slots --------

    def decay(self, slots: SlotDict, alpha: float = 0.9) -> None:
        """wkv <- wkv * alpha in place; token-shift untouched (wkvm's "decay")."""
        i = [int(slots["wkv"])]
        ops.slot_affine(self.wkv, 1, i, i, None, float(alpha))

    def merge(self, dst: SlotDict, a: SlotDict, b: SlotDict, weight: float = 0.5) -> None:
        """Every family: dst <- (1 - weight) * a + weight * b (wkvm's "merge")."""
        for fam, t, dim in (("wkv", self.wkv, 1), ("shift", self.shift, 2)):
            ops.slot_affine(t, dim, [int(dst[fam])], [int(a[fam])], [int(b[fam])],
                            1.0 - float(weight), float(weight))

    # -- decode -----------------------------------------------------------

    def wkv_decode(self, layer: int, slot_ids, r, w, k, v, kk, a) -> torch.Tensor:
        """One layer's WKV step for a batch, state updated in place."""
        return ops.wkv7_decode_slots(r, w, k, v, kk, a, self.wkv, layer, slot_ids)

    def device_ids(self, slot_batch: Sequence[SlotDict], family: str = "wkv") -> torch.Tensor:
        """Validated int32 device ids for a batch (reuse across layers/steps)."""
        return ops.slot_ids_tensor(_ids(slot_batch, family), self.num_slots + 1, self.device)

    # -- gather / scatter (wkvm/runner/state.py:63-97) ----------------------

    def gather_cache(self, slot_batch: Sequence[SlotDict], resident: bool | None = None):
        """wkvm's RWKV7StateBank.gather_cache: an fla ``Cache`` seeded with the
        batch's states (offset 0), for one model forward; commit it with
        :meth:`scatter_cache`. wkvm's RWKV7Runner calls the pair around every
        forward (wkvm/runner/runner.py:53-61, 79-87).

        ``resident`` (default: whether ``fla_compat.install()`` is in effect)
        picks what the cache holds. Resident: each layer's recurrent state is
        a :class:`~wkvm_b200.fla_compat.SlotState` that the installed ops
        update in place in ``wkv[layer, slot]``, and the token-shift rows are
        gathered by one kernel; nothing of the wkv family is copied. Not
        resident: plain tensor copies, as wkvm's bank gives them (one gather
        kernel per family for all layers), for fla's own ops or any caller
        that edits the states."""
        from fla.models.utils import Cache

        from . import fla_compat

        wkv_ids = _ids(slot_batch, "wkv")
        shift_ids = _ids(slot_batch, "shift")
        if resident is None:
            resident = fla_compat.installed()
        if resident:
            h = fla_compat.slot_cache(self, wkv_ids, shift_ids=shift_ids)
            h.cache._wkvm_slot_handle = h
            return h.cache
        wkv = ops.slot_gather_outer_major(self.wkv, 1, wkv_ids)      # [L, n, H, K, V]
        shift = ops.slot_gather_outer_major(self.shift, 2, shift_ids)  # [L, 2, n, D]
        cache = Cache()
        for i in range(self.layout.n_layer):
            cache.update(recurrent_state=wkv[i], conv_state=shift[i, 0], ffn_state=shift[i, 1],
                         layer_idx=i, offset=0)
        return cache

    def scatter_cache(self, slot_batch: Sequence[SlotDict], cache) -> None:
        """wkvm's RWKV7StateBank.scatter_cache: commits a forward's states
        back to the batch's rows. For a resident cache only the token-shift
        rows move (the wkv states were updated in place)."""
        handle = getattr(cache, "_wkvm_slot_handle", None)
        if handle is not None:
            handle.commit()
            return
        wkv_ids = _ids(slot_batch, "wkv")
        shift_ids = _ids(slot_batch, "shift")
        for i in range(self.layout.n_layer):
            st = cache[i]
            ops.slot_restore(self.wkv[i], 0, wkv_ids,
                             st["recurrent_state"].to(WKV_DTYPE).contiguous())
            ops.slot_restore(self.shift[i, 0], 0, shift_ids,
                             st["conv_state"].to(self.shift.dtype).contiguous())
            ops.slot_restore(self.shift[i, 1], 0, shift_ids,
                             st["ffn_state"].to(self.shift.dtype).contiguous())

    # -- snapshot / restore (wkvm/store.py:108-156) --------------------------

    def snapshot(self, slots: SlotDict) -> dict[str, torch.Tensor]:
        """Pinned host copies {"wkv": [L,H,K,V], "shift": [L,2,D]} — the
        tensors wkvm's StateStore.save keeps in its WARM tier. Synchronises."""
        wkv = ops.slot_snapshot(self.wkv, 1, [int(slots["wkv"])])
        shift = ops.slot_snapshot(self.shift, 2, [int(slots["shift"])])
        torch.cuda.current_stream(self.device).synchronize()
        return {"wkv": wkv[0], "shift": shift[0]}

    def snapshot_many(self, slot_batch: Sequence[SlotDict]) -> dict[str, torch.Tensor]:
        """Batched snapshot: {"wkv": [n,L,H,K,V], "shift": [n,L,2,D]} pinned."""
        wkv = ops.slot_snapshot(self.wkv, 1, _ids(slot_batch, "wkv"))
        shift = ops.slot_snapshot(self.shift, 2, _ids(slot_batch, "shift"))
        torch.cuda.current_stream(self.device).synchronize()
        return {"wkv": wkv, "shift": shift}

    def restore(self, slots: SlotDict, tensors: Mapping[str, torch.Tensor]) -> None:
        """Inverse of :meth:`snapshot` (wkvm StateStore.load). Synchronises."""
        # pinned copies stay alive until the kernels have read them
        wkv = _pinned(tensors["wkv"].reshape(1, *tensors["wkv"].shape))
        shift = _pinned(tensors["shift"].reshape(1, *tensors["shift"].shape))
        ops.slot_restore(self.wkv, 1, [int(slots["wkv"])], wkv)
        ops.slot_restore(self.shift, 2, [int(slots["shift"])], shift)
        torch.cuda.current_stream(self.device).synchronize()

    # -- migration --------------------------------------------------------

    def migrate_to(self, peer: "RWKV7StateBank", src: Sequence[SlotDict],
                   dst: Sequence[SlotDict]) -> torch.cuda.Event:
        """Copies slots to ``peer`` (another GPU's bank) with peer stores.
        Returns an event recorded after the copy on this GPU's stream; the
        source slots may be freed once it completes."""
        if peer.layout != self.layout:
            raise ValueError("peer bank has a different layout")
        ops.slot_migrate(self.wkv, peer.wkv, 1, _ids(src, "wkv"), _ids(dst, "wkv"))
        ops.slot_migrate(self.shift, peer.shift, 2, _ids(src, "shift"), _ids(dst, "shift"))
        ev = torch.cuda.Event()
        ev.record(torch.cuda.current_stream(self.device))
        return ev

    def state_bytes(self) -> int:
        return (self.wkv.numel() * self.wkv.element_size()
                + self.shift.numel() * self.shift.element_size())


@dataclass(frozen=True)
class SSMStateLayout:
    """Per-slot state shapes of selective state space layers: ``d_inner``
    channels of ``d_state`` states, and the last ``d_conv - 1`` inputs of the
    short convolution in the model's dtype."""

    n_layer: int
    d_inner: int
    d_state: int = 16
    d_conv: int = 4
    dtype: torch.dtype = torch.bfloat16

    def __post_init__(self) -> None:
        row = (self.d_conv - 1) * self.d_inner * torch.empty((), dtype=self.dtype).element_size()
        if row % 16 or self.d_inner * self.d_state % 4:
            raise ValueError("a slot's rows must be multiples of 16 bytes (the slot copies move whole vectors): "
                             f"{row} bytes of convolution inputs, {self.d_inner * self.d_state * 4} of states")

    @property
    def ssm_shape(self) -> tuple[int, int]:
        return (self.d_inner, self.d_state)

    @property
    def conv_shape(self) -> tuple[int, int]:
        return (self.d_conv - 1, self.d_inner)


class SSMStateBank:
    """Slot-indexed states of selective state space layers, with the slot
    operations zero, fork, snapshot and restore:

      ssm  [L, S+1, D, N] fp32          (slot 0 = reserved padding row)
      conv [L, S+1, W-1, D] model dtype (the last W-1 inputs, oldest first)

    ``conv`` / ``scan`` run one layer's short convolution and selective scan
    for a batch of slots (``decode`` for new tokens, ``prefill`` for prompts),
    states read and written in place."""

    FAMILIES = (("ssm", 1), ("conv", 1))  # (tensor, slot axis)

    def __init__(self, layout: SSMStateLayout, num_slots: int, device: torch.device | str = "cuda") -> None:
        self.layout = layout
        self.num_slots = num_slots
        self.device = torch.device(device)
        self.ssm = torch.zeros((layout.n_layer, num_slots + 1, *layout.ssm_shape), dtype=torch.float32,
                               device=self.device)
        self.conv = torch.zeros((layout.n_layer, num_slots + 1, *layout.conv_shape), dtype=layout.dtype,
                                device=self.device)

    def device_ids(self, slots: Sequence[int]) -> torch.Tensor:
        """Validated int32 device ids for a batch (reuse across layers/steps)."""
        return ops.slot_ids_tensor(slots, self.num_slots + 1, self.device)

    # -- one layer --------------------------------------------------------

    def conv_decode(self, layer: int, slot_ids, x, weight, bias=None, activation="silu") -> torch.Tensor:
        return ssm.short_conv_decode_slots(x, weight, self.conv, layer, slot_ids, bias=bias, activation=activation)

    def conv_prefill(self, layer: int, slot_ids, x, weight, bias=None, activation="silu",
                     cu_seqlens=None) -> torch.Tensor:
        return ssm.short_conv_prefill_slots(x, weight, self.conv, layer, slot_ids, bias=bias, activation=activation,
                                            cu_seqlens=cu_seqlens)

    def scan_decode(self, layer: int, slot_ids, x, dt, A, B, C, **more) -> torch.Tensor:
        """``more``: D, z, dt_bias, dt_softplus of :func:`~wkvm_b200.ssm.selective_scan`."""
        return ssm.selective_scan_decode_slots(x, dt, A, B, C, self.ssm, layer, slot_ids, **more)

    def scan_prefill(self, layer: int, slot_ids, x, dt, A, B, C, cu_seqlens=None, **more) -> torch.Tensor:
        return ssm.selective_scan_prefill_slots(x, dt, A, B, C, self.ssm, layer, slot_ids, cu_seqlens=cu_seqlens,
                                                **more)

    # -- slot lifecycle ---------------------------------------------------

    def zero(self, slots: Sequence[int]) -> None:
        for name, dim in self.FAMILIES:
            ops.slot_zero(getattr(self, name), dim, slots)

    def fork(self, parents: Sequence[int], children: Sequence[int]) -> None:
        for name, dim in self.FAMILIES:
            ops.slot_copy(getattr(self, name), dim, parents, children)

    def snapshot(self, slots: Sequence[int]) -> dict[str, torch.Tensor]:
        """Pinned host copies {"ssm": [n, L, D, N], "conv": [n, L, W-1, D]}. Synchronises."""
        got = {name: ops.slot_snapshot(getattr(self, name), dim, slots) for name, dim in self.FAMILIES}
        torch.cuda.current_stream(self.device).synchronize()
        return got

    def restore(self, slots: Sequence[int], tensors: Mapping[str, torch.Tensor]) -> None:
        """Inverse of :meth:`snapshot`. Synchronises."""
        staged = [_pinned(tensors[name]) for name, _ in self.FAMILIES]  # alive until the kernels have read them
        for (name, dim), t in zip(self.FAMILIES, staged):
            ops.slot_restore(getattr(self, name), dim, slots, t)
        torch.cuda.current_stream(self.device).synchronize()

    def state_bytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.ssm, self.conv))


def _pinned(t: torch.Tensor) -> torch.Tensor:
    if t.is_cuda:
        return t.contiguous()
    t = t.contiguous()
    return t if t.is_pinned() else t.pin_memory()
