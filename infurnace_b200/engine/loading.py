"""From a model folder to a runner: configuration, plan, weights, parts, cache."""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from ..cache import CacheLayout, CacheManager
from ..errors import ModelConfigError
from ..config.specs import AttentionSpec, DenseMLPSpec, GatedMLPSpec, KVCacheNeed, PagedCacheNeed
from ..kernels.low_bits import kv8_room_bytes
from ..models import plan_for, read_config
from ..parts import DecoderModel, Runtime
from ..weights.loader import load_weights
from .runner import ModelRunner

DTYPES = {"bfloat16": torch.bfloat16, "bf16": torch.bfloat16, "float32": torch.float32, "fp32": torch.float32}


@dataclass
class EngineOptions:
    """How much of the device an engine may use; none of these is a property of the model."""
    dtype: str = "bfloat16"
    device: str = "cuda"
    page_size: int = 16
    num_pages: Optional[int] = None            # pages of each key/value group
    max_num_seqs: int = 8                      # live requests (state slots)
    max_num_batched_tokens: int = 2048         # tokens of one step
    max_model_len: Optional[int] = None        # longest sequence; default: the model's limit
    memory_fraction: float = 0.8               # of free device memory, when num_pages is None
    weight_format: str = "stored"              # "mx4": attention and dense feed-forward matrices in microscaled 4-bit floating point
    cache_format: str = "dtype"                # "int8": keys and values in 8 bits with a scale for each page and head

    def check_formats(self):
        if self.weight_format not in ("stored", "mx4"):
            raise ModelConfigError(f"weight_format {self.weight_format!r}: choose stored or mx4")
        if self.cache_format not in ("dtype", "int8"):
            raise ModelConfigError(f"cache_format {self.cache_format!r}: choose dtype or int8")
        if self.cache_format == "int8" and (self.page_size % 16 or not 16 <= self.page_size <= 4096):
            raise ModelConfigError(f"cache_format int8 wants pages of a multiple of 16 tokens up to 4,096, not {self.page_size}")


def parse_dtype(name):
    if isinstance(name, torch.dtype):
        return name
    try:
        return DTYPES[name]
    except KeyError:
        raise ModelConfigError(f"dtype {name!r}: choose bfloat16 or float32") from None


def build_runner(model_dir: Optional[str], options: EngineOptions, kernels=None, progress=None, random=None):
    """(config, plan, runner) for the model folder.  ``kernels`` None loads the CUDA kernel
    set, which fails loudly without a GPU or a compiler; tests may pass a stand-in.

    ``random`` = (config, seed, store_dtype name): no folder is read; the tensors are drawn on the
    device as the parts ask for them (weights/random_init.py), which is how models too large to pass
    through a file get their random weights."""
    dtype = parse_dtype(options.dtype)
    options.check_formats()
    config = read_config(model_dir) if random is None else random[0]
    plan = plan_for(config)
    check_plan(plan, options)
    if kernels is None:
        from ..kernels import load_cuda_kernels
        kernels = load_cuda_kernels(progress=progress)
    runtime = Runtime(device=torch.device(options.device), act_dtype=dtype, kernels=kernels,
                      weight_format=options.weight_format)
    if random is None:
        weights = load_weights(model_dir, plan, dtype, runtime.device, progress=progress)
    else:
        from ..weights.random_init import DeviceRandomWeights
        weights = DeviceRandomWeights(plan, random[1], dtype, runtime.device, kernels, store_dtype=parse_dtype(random[2]))
    model = DecoderModel(plan, weights, runtime)
    del weights
    runtime.share_row_room(max(options.max_num_batched_tokens, options.max_num_seqs))
    max_len = min(options.max_model_len or plan.max_positions, plan.max_positions)
    num_pages = options.num_pages
    if num_pages is None:
        num_pages = default_num_pages(plan, options, dtype, runtime.device, max_len)
    room = room_bytes(plan, options, dtype, max_len, num_pages) if getattr(kernels, "attention_tc", False) else 0
    cache = CacheManager(plan, options.page_size, num_pages, options.max_num_seqs, dtype=dtype, device=runtime.device,
                         cache_format=options.cache_format, room_bytes=room)
    runner = ModelRunner(model, cache, runtime, options.max_num_batched_tokens, max_len)
    return config, plan, runner


def check_plan(plan, options) -> None:
    """Refuse formats that a model's parts do not have, before anything is loaded.  4 bits: attention and dense feed-forwards,
    whose every width is a multiple of 32 (other parts' matrices stay as stored, but a model without any such part is refused).
    8-bit pages: every mixer that keeps keys and values is plain grouped-query attention with heads of a multiple of 16."""
    def parts(layer):
        return [x for x in (getattr(layer, "mixer", None), getattr(layer, "ffn", None)) if x is not None]
    if options.weight_format == "mx4":
        widths = []
        for part in (p for layer in plan.layers for p in parts(layer)):
            if isinstance(part, AttentionSpec):
                widths += [part.hidden_size, part.num_heads * part.head_dim]
            elif isinstance(part, (GatedMLPSpec, DenseMLPSpec)):
                widths += [part.hidden_size, part.intermediate_size]
        if not widths:
            raise ModelConfigError("weight_format mx4: the model has neither grouped-query attention nor a dense feed-forward")
        if any(w % 32 for w in widths):
            raise ModelConfigError(f"weight_format mx4: widths are multiples of 32, not {sorted({w for w in widths if w % 32})}")
    if options.cache_format == "int8":
        for call in plan.resolved_schedule():
            layer = plan.layers[call.layer]
            need = layer.cache_need()
            for sub in need if isinstance(need, tuple) else (need,):
                if isinstance(sub, (KVCacheNeed, PagedCacheNeed)):
                    mixer = getattr(layer, "mixer", None)
                    if not isinstance(mixer, AttentionSpec):
                        raise ModelConfigError(f"cache_format int8: {type(mixer or layer).__name__} reads its pages in the engine's dtype")
                    if mixer.head_dim % 16 or not 16 <= mixer.head_dim <= 256:
                        raise ModelConfigError(f"cache_format int8: head_dim is a multiple of 16 up to 256, not {mixer.head_dim}")


def room_bytes(plan, options, dtype, max_len, num_pages) -> int:
    """Bytes of the room for expanded 8-bit pages that an engine's layers share (``num_pages``: as in the cache manager)."""
    if options.cache_format != "int8":
        return 0
    each = -(-max_len // options.page_size)
    return max((kv8_room_bytes(num_pages[key] if isinstance(num_pages, dict) else num_pages, options.max_num_seqs, each,
                               need.streams[0].heads, options.page_size, need.streams[0].width, dtype)
                for key, (need, _) in CacheLayout(plan).kv.items()), default=0)


def default_num_pages(plan, options, dtype, device, max_len) -> int:
    """Pages for ``max_num_seqs`` sequences of ``max_model_len``, capped by the share of
    free device memory that ``memory_fraction`` allows, the room for expanded 8-bit pages counted."""
    layout = CacheLayout(plan)
    per_page = 0
    esize = 1 if options.cache_format == "int8" else torch.empty((), dtype=dtype).element_size()
    for need, ids in layout.kv.values():
        per_page += len(ids) * sum(x.heads * x.width for x in need.streams) * options.page_size * esize
    want = options.max_num_seqs * (-(-max_len // options.page_size)) + 1
    if per_page == 0:
        return 1
    if device.type == "cuda":
        free, _ = torch.cuda.mem_get_info(device)
        free = int(free * options.memory_fraction)
        room = [room_bytes(plan, options, dtype, max_len, n) for n in (0, 1, want)]
        fit = max((free - room[2]) // per_page, (free - room[0]) // (per_page + room[1] - room[0]))
        want = max(1, min(want, fit))
    return want
