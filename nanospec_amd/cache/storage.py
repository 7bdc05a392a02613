"""The memory behind the cache manager: pages of keys and values per group of layers, and state slots.

A run-order entry of the model with a ``PagedNeed`` gets one layer of its group's page tensors:
    K [entries, pages, kv_heads, page, head_dim]       (the reference keeps [pages, page, kv_heads, head_dim],
                                                        kv/cache.py:16-19; here a head's part of a page is contiguous)
    V [entries, pages, kv_heads, value_dim, page]      (transposed per page for the attention kernels; value_dim is
                                                        head_dim unless the mixer says otherwise)
or, with ``kv_format="int4"``, one of its pages of 4 bits [entries, pages, kv_heads, page / 8, record] (``kernels.ops.Kv4Pages``).
All start as zeros: slots that are masked out are still read (reference: kv/cache.py:18).  A page id
means the same page in every entry of its group.  An entry with a ``StateNeed`` gets a tensor
[slots, *shape]; an entry that reads another entry's cache gets that entry's view.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from ..kernels.ops import Kv4Pages, SlotTensors, kv4_read, kv4_takes
from ..parts.needs import PagedNeed, StateNeed, each_need
from .manager import GroupSpec


KV_FORMATS = ("model", "int4")  # keys and values in the model's precision, or in 4 bits with a step and a lowest value for each token and head
STEPS_SHARE = 0.1  # of the device's memory that is to be left for the steps beside weights, pages and states


@dataclass
class PagedView:
    group: int
    k: torch.Tensor
    v: torch.Tensor


@dataclass
class Int4View:
    group: int
    pages: Kv4Pages
    products: dict  # of all of the storage's entries: mixer -> the product that it runs over this cache (others run their own)


@dataclass
class StateView:
    state: torch.Tensor  # [slots, *shape]


def plan_groups(cache_needs: list) -> tuple[list[GroupSpec], list[PagedNeed], list[int | None]]:
    """Run-order entries with equal paged needs share a group.  -> (group specs for the manager, the need
    of each group, group index of each entry or None)."""
    needs: list[PagedNeed] = []
    of_entry: list[int | None] = []
    for need in cache_needs:
        if isinstance(need, PagedNeed):
            if need not in needs:
                needs.append(need)
            of_entry.append(needs.index(need))
        else:
            # (an entry whose mixer is made of several: its paged needs join their groups; ``of_entry`` names the first)
            first = None
            for single in each_need(need) if isinstance(need, (tuple, list)) else ():
                if isinstance(single, PagedNeed):
                    if single not in needs:
                        needs.append(single)
                    first = needs.index(single) if first is None else first
            of_entry.append(first)
    specs = [GroupSpec(n.group_name, n.window) for n in needs]
    return specs, needs, of_entry


def check_int4(model, page_size: int) -> None:
    """Whether every entry of the model's run order that keeps or reads keys and values does so in 4 bits too, with pages of ``page_size`` tokens."""
    for i, (need, call) in enumerate(zip(model.cache_needs, model.spec.run_order)):
        if call.cache_from is not None:
            need = model.cache_needs[call.cache_from]
            if not getattr(getattr(model.layers[call.layer], "mixer", None), "takes_int4_cache", False):
                raise ValueError(f"entry {i} of the run order reads another entry's keys and values and does not do so in 4 bits")
        for single in each_need(need):
            if isinstance(single, PagedNeed) and not single.int4:
                raise ValueError(f"entry {i} of the run order does not keep its keys and values in 4 bits: that is built for soft-max attention over rotated keys with values of the keys' size, "
                                 "without gates, sinks, caps, biases or norms of its own")
            if isinstance(single, PagedNeed) and not kv4_takes(single.head_dim, page_size):
                raise ValueError(f"keys and values in 4 bits take heads of a multiple of 32 channels up to 256 and pages of a power of two of tokens from 8, not {single.head_dim} channels and "
                                 f"pages of {page_size}")


class CacheStorage:
    def __init__(self, model, num_pages: list[int], page_size: int, num_slots: int, dtype, device, kv_format: str = "model") -> None:
        if kv_format not in KV_FORMATS:
            raise ValueError(f"kv_format={kv_format!r}: use one of {KV_FORMATS}")
        self.kv_format = kv_format
        self.products: dict = {}
        if kv_format == "int4":
            check_int4(model, page_size)
        # what a model keeps only to be faster makes room, and what its layers would have for a cache in 4 bits: where the pages do not fit beside it, or leave little for the steps
        give_back = getattr(model, "give_back_second_copies", lambda: False)
        short = False
        try:
            if kv_format == "int4":
                self.products = model.serve_int4_cache() or {}
            self._allocate(model, num_pages, page_size, num_slots, dtype, device)
        except torch.OutOfMemoryError:
            short = True
        if short:  # (behind the handler, whose traceback holds what had been allocated)
            products = self.products
            self.__dict__.clear()
            self.kv_format, self.products = kv_format, products
            self._one_order(model)
            give_back()
            self._allocate(model, num_pages, page_size, num_slots, dtype, device)
        elif (dtype == torch.float32 or self.products) and torch.device(device).type == "cuda":  # (no other models have such copies)
            free, total = torch.cuda.mem_get_info(device)
            if free + torch.cuda.memory_reserved(device) - torch.cuda.memory_allocated(device) < STEPS_SHARE * total:
                self._one_order(model)
                give_back()

    def _one_order(self, model) -> None:
        if self.kv_format == "int4" and getattr(model, "stream_one_order", lambda products: False)(self.products):
            self.products.clear()  # (the views' too: the layers' own products are those)

    def _allocate(self, model, num_pages: list[int], page_size: int, num_slots: int, dtype, device) -> None:
        self.group_specs, needs, of_entry = plan_groups(model.cache_needs)
        self.page_size = page_size
        flat = [(single, i) for i, (need, call) in enumerate(zip(model.cache_needs, model.spec.run_order)) if call.cache_from is None
                for single in each_need(need)]
        counts = [sum(1 for single, _ in flat if isinstance(single, PagedNeed) and needs.index(single) == i) for i in range(len(needs))]
        int4 = self.kv_format == "int4"
        self.k = [] if int4 else [torch.zeros((counts[i], num_pages[i], n.kv_heads, page_size, n.head_dim), dtype=dtype, device=device)
                                  for i, n in enumerate(needs)]
        self.v = [] if int4 else [torch.zeros((counts[i], num_pages[i], n.kv_heads, n.v_dim, page_size), dtype=dtype, device=device)
                                  for i, n in enumerate(needs)]
        self.int4 = [torch.zeros((counts[i], *Kv4Pages.shape(num_pages[i], n.kv_heads, page_size, n.head_dim)), dtype=torch.uint8, device=device)
                     for i, n in enumerate(needs)] if int4 else []
        self.states: list[torch.Tensor] = []
        self.views: list = []
        taken = [0] * len(needs)
        def view_of(need):
            if isinstance(need, (tuple, list)):
                return tuple(view_of(single) for single in need)
            if isinstance(need, PagedNeed):
                g = needs.index(need)
                view = Int4View(g, Kv4Pages(self.int4[g][taken[g]], need.head_dim), self.products) if int4 else PagedView(g, self.k[g][taken[g]], self.v[g][taken[g]])
                taken[g] += 1
                return view
            if isinstance(need, StateNeed):
                t = torch.zeros((num_slots, *need.shape), dtype=need.dtype, device=device)
                self.states.append(t)
                return StateView(t)
            return None

        for i, (need, call) in enumerate(zip(model.cache_needs, model.spec.run_order)):
            self.views.append(self.views[call.cache_from] if call.cache_from is not None else view_of(need))
        # state that belongs to the model and to no layer (``model.state_needs``: name -> StateNeed)
        self.model_state: dict[str, torch.Tensor] = {}
        for name, need in getattr(model, "state_needs", {}).items():
            t = torch.zeros((num_slots, *need.shape), dtype=need.dtype, device=device)
            self.states.append(t)
            self.model_state[name] = t
        # (a single state is as fast through its own fill, and the CPU has no launches to save)
        self._slots = SlotTensors(self.states) if len(self.states) > 1 and torch.device(device).type == "cuda" else None

    def reset_slot(self, slot: int) -> None:
        """A newly admitted request starts from zero state."""
        if self._slots is not None:
            self._slots.clear(slot)
            return
        for t in self.states:
            t[slot].zero_()

    def kept(self, entry: int, positions: torch.Tensor, token_req: torch.Tensor, block_table: torch.Tensor):
        """-> (keys, values) [tokens, kv_heads, size], float32, of the tokens at ``positions`` of requests ``token_req`` as run-order entry ``entry`` keeps them (keys as the scores meet them);
        ``block_table`` int32 [requests, pages] of the entry's group.  For looking at a cache: on the current stream, into new tensors."""
        view = self.views[entry]
        if isinstance(view, Int4View):
            return kv4_read(view.pages, positions, token_req, block_table, dtype=torch.float32)
        if not isinstance(view, PagedView):
            raise ValueError(f"entry {entry} of the run order keeps no keys and values in pages of its own")
        page, at = block_table[token_req.long(), positions.long() // self.page_size].long(), positions.long() % self.page_size
        return view.k[page, :, at].float(), view.v[page, :, :, at].float()

    def bytes_per_token(self) -> int:
        if self.kv_format == "int4":  # (records of eight tokens)
            return sum(t.shape[0] * t.shape[2] * t.shape[4] // 8 for t in self.int4)
        return sum((k[:, 0, :, 0].numel() + v[:, 0, :, :, 0].numel()) * k.element_size() for k, v in zip(self.k, self.v))
