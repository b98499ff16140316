"""Model registry: config.json's "architecture" picks the loader, as `llama_model_lookup` picks a LLaMA size from
a checkpoint.  A loader returns an object the Engine can serve (state_specs / vocab / dtype / device /
forward_portion)."""
import contextlib
import copy
import json
import os
import weakref
from typing import Callable, Dict, Optional

import torch

_LOADERS: Dict[str, Callable] = {}


def register(architecture: str):
    def deco(fn: Callable) -> Callable:
        _LOADERS[architecture] = fn
        return fn
    return deco


def architectures():
    return sorted(_LOADERS)


@register("Lugovik")
def _load_lugovik(model_dir: str, dtype: torch.dtype, device: torch.device, max_positions: int, config: dict):
    from . import lugovik

    return lugovik.load(model_dir, dtype=dtype, device=device, max_positions=max_positions)


@register("Zenasun")
def _load_zenasun(model_dir: str, dtype: torch.dtype, device: torch.device, max_positions: int, config: dict):
    from . import zenasun

    return zenasun.load(model_dir, dtype=dtype, device=device, max_positions=max_positions)


@register("Zuvevik")
def _load_zuvevik(model_dir: str, dtype: torch.dtype, device: torch.device, max_positions: int, config: dict):
    from . import zuvevik

    return zuvevik.load(model_dir, dtype=dtype, device=device, max_positions=max_positions)


@register("Rinirax")
def _load_rinirax(model_dir: str, dtype: torch.dtype, device: torch.device, max_positions: int, config: dict):
    from . import rinirax

    return rinirax.load(model_dir, dtype=dtype, device=device, max_positions=max_positions)


@register("Lukupel")
def _load_lukupel(model_dir: str, dtype: torch.dtype, device: torch.device, max_positions: int, config: dict):
    from . import lukupel

    return lukupel.load(model_dir, dtype=dtype, device=device, max_positions=max_positions)


@register("Malulorn")
def _load_malulorn(model_dir: str, dtype: torch.dtype, device: torch.device, max_positions: int, config: dict):
    from . import malulorn

    return malulorn.load(model_dir, dtype=dtype, device=device, max_positions=max_positions)


@register("LLaMA")
def _load_llama(model_dir: str, dtype: torch.dtype, device: torch.device, max_positions: int, config: dict):
    """config.json: {"architecture": "LLaMA", "name": "7B" | sizes..., "quantize": null | "gptq.int4" | ..., "checkpoint": file,
    "kv_cache": {"pages", "page", "store", "window", "first"}}: with "kv_cache" the arguments of `PagedLLaMAModel`, without it `LLaMASequenceModel`."""
    from .model import LLaMA, LLaMAConfig
    from .utils import EmptyInitOnDevice, lazy_load

    if dtype != torch.bfloat16:
        raise RuntimeError("the LLaMA path runs in bfloat16 only")
    cfg = LLaMAConfig.from_name(config["name"]) if "name" in config else LLaMAConfig(
        **{k: config[k] for k in ("block_size", "vocab_size", "n_layer", "n_head", "n_embd") if k in config})
    with EmptyInitOnDevice(device=device, dtype=torch.bfloat16, quantization_mode=config.get("quantize")):
        model = LLaMA(cfg)
    with lazy_load(os.path.join(model_dir, config.get("checkpoint", "lit-llama.pth"))) as sd:
        model.load_state_dict(sd)
    if "kv_cache" in config:
        return PagedLLaMAModel(model.eval(), max_positions=max_positions, **config["kv_cache"])
    return LLaMASequenceModel(model.eval(), max_positions or cfg.block_size)


class LLaMASequenceModel:
    """The package's LLaMA behind the Engine's model interface.  Its KV cache lives inside the module (one sequence
    at a time), so it declares no pooled state; a portion that starts at position 0 resets the cache."""
    graph_safe = False     # LLaMA.forward replays its own decode graph

    def __init__(self, model, max_seq_length: int) -> None:
        self.model, self.max_seq_length = model, int(max_seq_length)
        self.vocab = model.config.padded_vocab_size
        self.dtype = torch.bfloat16
        self.device = next(model.parameters()).device
        self._pos = 0

    def state_specs(self):
        return {}

    @torch.no_grad()
    def forward_portion(self, tokens: torch.Tensor, ctx, want: Optional[torch.Tensor] = None) -> torch.Tensor:
        pos0 = int(ctx.meta[1])
        if pos0 == 0:
            self.model.reset_cache()
        T = tokens.numel()
        input_pos = torch.arange(pos0, pos0 + T, device=tokens.device)
        logits = self.model(tokens.view(1, -1).to(torch.int64), self.max_seq_length, input_pos)[0]
        return (logits if want is None else logits.index_select(0, want.to(torch.int64))).float()


def _release_all(pages, owner) -> None:
    for request_id in [r for r in pages.requests() if isinstance(r, tuple) and r and r[0] is owner]:
        pages.release(request_id)


class PagedLLaMAModel:
    """The package's LLaMA behind the Engine's model interface with its keys and values in pages (paged.py), in bf16, e4m3 or int8: as many sequences at a
    time as there are slots, each with the pages that its length needs.  A model of MHA layers: every head has keys and values of its own.

    `pages` of `page` tokens are shared by the sequences (as many again for every layer).  The engine's scheduler lets a request wait until there are pages
    for all of it; a portion that finds none left raises PagesFull (a PoolFull), and the sequence stands where it stood.  With `window` a
    token sees the last `window` positions and the first `first` ones, and a sequence keeps no pages for the others, so it may grow without end; else
    it may have `max_positions` (default: the model's block size)."""
    graph_safe = False     # pages are booked on the host

    def __init__(self, model, *, pages: int, page: int = 64, store: str = "act", window: int = 0, first: int = 0, max_positions: int = 0) -> None:
        from .paged import PagedCache, PagePool

        cfg = model.config
        if model.transformer.wte.weight.dtype != torch.bfloat16:
            raise RuntimeError(f"wte dtype {model.transformer.wte.weight.dtype} unsupported; the model must be bf16 (model.to(torch.bfloat16))")
        self.model, self.vocab, self.dtype = model, cfg.padded_vocab_size, torch.bfloat16
        self.device = next(model.parameters()).device
        self.heads, self.size = cfg.n_head, cfg.n_embd // cfg.n_head
        self.window, self.first = int(window), int(first)
        self.max_positions = int(max_positions) or (0 if window else cfg.block_size)
        self.pages = PagePool(pages, page, self.device, window=self.window, first=self.first)
        self.caches = [PagedCache.empty(pages, page, self.heads, self.size, dtype=self.dtype, store=store, device=self.device) for _ in range(cfg.n_layer)]
        self.freq = (1.0 / 10000 ** (torch.arange(0, self.size, 2, dtype=torch.float32) / self.size)).to(self.device)
        self._owner = object()                              # whose slots these are: the model's own, or an engine's

    def for_engine(self) -> "PagedLLaMAModel":
        """The same weights and pages with slots of its own, which an engine has: engines that share a model number their slots alike.  Pages of an engine that is
        gone are free.  Pages that one gives back another takes, so engines that share a model run on one stream."""
        view = copy.copy(self)
        view._owner = object()
        weakref.finalize(view, _release_all, self.pages, view._owner).atexit = False
        return view

    def state_specs(self):
        return {}

    def release_slot(self, slot: int) -> None:
        """The engine's slot is free: so are its sequence's pages."""
        if self.pages.has((self._owner, slot)):
            self.pages.release((self._owner, slot))

    def book(self, slot: int, pos0: int, n: int):
        """The step of a slot's next n tokens, at position pos0 of its sequence; a slot at position 0 begins a new one."""
        if pos0 == 0:
            self.release_slot(slot)
        elif not self.pages.has((self._owner, slot)) or self.pages.position((self._owner, slot)) != pos0:
            raise RuntimeError(f"paged LLaMA: slot {slot} is not at position {pos0}")
        return self.pages.step([((self._owner, slot), n)])

    @contextlib.contextmanager
    def booked(self, slot: int, pos0: int, n: int):
        """The same for what runs inside: if it raises, the slot's sequence stands where it stood."""
        step = self.book(slot, pos0, n)
        try:
            yield step
        except BaseException:
            self.pages.take_back((self._owner, slot), n)
            raise

    def has_room(self, live, tokens: int, portion: int) -> bool:
        """Whether one more sequence, of `tokens` tokens, finds pages beside those of `live` (slot -> the tokens that its sequence grows to), fed at most
        `portion` tokens at a time."""
        def most(n: int) -> int:
            return min(n, self.max_positions) if self.max_positions else n

        return self.pages.has_room({(self._owner, slot): most(n) for slot, n in live.items()}, most(tokens), portion)

    def _rotated(self, x: torch.Tensor, ctx) -> torch.Tensor:
        """Every head of x [T, heads * size] (rows of a wider product) turned by position, pairs of neighbouring entries (lit_llama/model.py:306-323)."""
        from . import _seqlib as S

        T, n = x.shape
        out = torch.empty((T, self.heads, self.size), dtype=x.dtype, device=x.device)
        S.check(S.lib().b2l_seq_rope(S.ptr(x), x.stride(0), 0, S.ptr(self.freq), self.size, 1, 0, 1.0, 1.0, S.ptr(ctx.meta), S.ptr(out), n, 0, T, self.heads, self.size, self.size,
                                     self.size, ctx.act, ctx.stream), "b2l_seq_rope")
        return out

    @torch.no_grad()
    def forward_portion(self, tokens: torch.Tensor, ctx, want: Optional[torch.Tensor] = None) -> torch.Tensor:
        slot, pos0 = (ctx.slot_hint, ctx.pos_hint) if ctx.slot_hint is not None else ctx.meta.tolist()
        with self.booked(slot, pos0, tokens.numel()) as step:
            return self._portion(tokens, ctx, want, step)

    def _portion(self, tokens: torch.Tensor, ctx, want: Optional[torch.Tensor], step) -> torch.Tensor:
        from . import _lib as L
        from .model import _add

        T, C = tokens.numel(), self.heads * self.size
        tokens = tokens.to(torch.int64).contiguous()
        wte = self.model.transformer.wte.weight
        x = torch.empty((1, T, C), dtype=self.dtype, device=self.device)
        L.check(L.lib().b2l_embedding(tokens.data_ptr(), 1, wte.data_ptr(), x.data_ptr(), T, C, wte.shape[0], L.stream_ptr()), "b2l_embedding")
        for block, cache in zip(self.model.transformer.h, self.caches):
            qkv = block.attn.c_attn(block.rms_1(x))[0]
            cache.write(self._rotated(qkv[:, C:2 * C], ctx), qkv[:, 2 * C:].unflatten(1, (self.heads, self.size)), step)
            att = cache.attend(self._rotated(qkv[:, :C], ctx), step, window=self.window, first=self.first)
            x = _add(x, block.attn.c_proj(att.view(1, T, C)))
            x = _add(x, block.mlp(block.rms_2(x)))
        if want is not None:
            x = x.index_select(1, want.to(torch.int64))
        if x.shape[1] == 0:
            return torch.empty((0, self.vocab), dtype=torch.float32, device=self.device)
        return self.model.lm_head(self.model.transformer.ln_f(x))[0].float()


def read_config(model_dir: str) -> dict:
    with open(os.path.join(model_dir, "config.json")) as f:
        return json.load(f)


def load_model(model_dir: str, dtype: torch.dtype = torch.bfloat16, device: Optional[torch.device] = None, max_positions: int = 0):
    """The model of `model_dir` (config.json + weights) on `device`, chosen by config.json's architecture."""
    config = read_config(model_dir)
    arch = config.get("architecture")
    if arch not in _LOADERS:
        raise ValueError(f"unknown architecture {arch!r}; registered: {architectures()}")
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    return _LOADERS[arch](model_dir, dtype, device, max_positions, config)
