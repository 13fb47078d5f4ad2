"""Autoregressive sampling from a ratchet model (drop-in for ``generate.py``).

Same public functions as the reference (``generate.py:38-206``): ``load_for_generation``
rebuilds a model from a checkpoint's metadata and safetensors (``model::``-prefixed keys,
``checkpoint.py:23-60``), ``warm_up_generation`` and ``generate``.

What differs is how a token is produced. The reference runs the whole (padded) window
through the model for every new token and reads the logits at the last real position
(``generate.py:183-201``). Here the window is run once (``RatchetGPT.prefill``) and each
new token is one step over a KV cache (``RatchetGPT.decode_step``): M = batch rows through
every ratchet GEMM, which dispatches to the small-M int8 kernel. Attention is causal, so
the last position's logits are the same quantity the full-window forward computes (equal
up to float summation order). Past ``block_size`` tokens the reference re-positions a
sliding window every step; positions are absolute, so a cache cannot follow, and this
module then recomputes the window each step exactly as the reference does.
"""

from __future__ import annotations

import json
from pathlib import Path
from typing import Literal

import torch
from torch import Tensor

from .decode import decode_greedy, reserve_step
from .model import Int8KVCache, KVCache, ModelConfig, RatchetGPT, build_seeded_model
from .ratchet import DiscreteRatchetLinear


# The architecture fields a checkpoint's experiment config carries, with their types; the
# rest of the model config is fixed for generation (no dropout) or derived (vocabulary).
_ARCHITECTURE = (("block_size", int), ("n_layer", int), ("n_head", int), ("n_embd", int))
_OPTIONAL = (("matmul_mode", str, "fp32"), ("ratchet_embedding", bool, False),
             ("rms_ema_beta", float, 0.0), ("pressure_leak_period", int, 0),
             ("attention_softcap", float, 0.0), ("distance_bias", bool, False))


def _checkpoint_files(base_path: str | Path) -> tuple[Path, Path]:
    """(metadata .json, tensors .safetensors) of a checkpoint named by its stem or by
    either file (``checkpoint.py:23-60`` writes the pair side by side)."""
    stem = Path(base_path)
    if stem.suffix in (".json", ".safetensors"):
        stem = stem.with_suffix("")
    return stem.with_suffix(".json"), stem.with_suffix(".safetensors")


def _model_config(metadata: dict) -> ModelConfig:
    """The ModelConfig a checkpoint was trained with: every buffer the model registers
    (e.g. ``rms_ema`` when its beta is positive) must exist before the strict load."""
    if metadata.get("tokenizer_kind", "char") != "char":
        raise ValueError("only character-vocabulary checkpoints are supported")
    stored = metadata["experiment_config"]
    fields = {name: kind(stored[name]) for name, kind in _ARCHITECTURE}
    fields.update({name: kind(stored.get(name, default)) for name, kind, default in _OPTIONAL})
    if stored.get("ffn_hidden") is not None:
        fields["ffn_hidden"] = int(stored["ffn_hidden"])
    return ModelConfig(vocab_size=len(metadata["vocabulary"]), dropout=0.0, **fields)


def load_for_generation(
    base_path: str | Path,
    *,
    device: str | torch.device = "cpu",
    inference_matmul_mode: Literal["checkpoint", "fp32", "bf16", "int8"] = "checkpoint",
) -> tuple[RatchetGPT, tuple[str, ...]]:
    """Rebuild a model from its checkpoint (eval mode) and return it with its vocabulary
    (char checkpoints; ``generate.py:38-92``). ``inference_matmul_mode`` other than
    "checkpoint" switches every ratchet layer to that matmul path after loading."""
    from safetensors.torch import load_file

    meta_file, tensor_file = _checkpoint_files(base_path)
    metadata = json.loads(meta_file.read_text())
    config = _model_config(metadata)
    # max_code 0 is the float control arm (plain linears)
    model = build_seeded_model(config, max_code=int(metadata["max_code"]) or None, seed=0)
    prefix = "model::"
    model.load_state_dict({key[len(prefix):]: tensor
                           for key, tensor in load_file(tensor_file).items()
                           if key.startswith(prefix)}, strict=True)
    for layer in _ratchet_layers(model):
        if inference_matmul_mode != "checkpoint":
            layer.matmul_mode = inference_matmul_mode
    return model.to(device).eval(), tuple(metadata["vocabulary"])


def _ratchet_layers(model: RatchetGPT) -> list[DiscreteRatchetLinear]:
    return [m for m in model.modules() if isinstance(m, DiscreteRatchetLinear)]


@torch.no_grad()
def warm_up_generation(model: RatchetGPT, *, device: str | torch.device | None = None) -> bool:
    """Touch the int8 decode path once before timing (``generate.py:117-132``): a one-token
    prefill and one cached step on a scratch cache, the two kernels sequences ``generate``
    runs. The HIP kernels are compiled ahead of time, so nothing is built per shape; this
    only pays the library's first-launch costs. Returns whether anything ran (models
    without int8 layers need no warm-up)."""
    if not any(layer.matmul_mode == "int8" for layer in _ratchet_layers(model)):
        return False
    where = torch.device(device) if device is not None else next(model.parameters()).device
    scratch = model.new_cache(1, max_len=min(2, model.config.block_size))
    token = torch.zeros((1, 1), dtype=torch.long, device=where)
    model.prefill(token, scratch)
    if scratch.length < scratch.max_len:
        model.decode_step(token, scratch)
    if where.type == "cuda":
        torch.cuda.synchronize(where)
    return True


class DecodeGraph:
    """One decode step captured as a HIP graph and replayed: the token ids go into a fixed
    device buffer, the position is the cache's device tensor, and the logits come back in a
    fixed buffer. Replay does exactly the work of ``RatchetGPT.decode_step``.

    With ``greedy=True`` the graph also takes each row's argmax into `tokens` and advances
    the cache position (``decode.decode_greedy``): replays then chain greedy steps on the
    device (``next_greedy``), the reference's temperature-0 loop (``generate.py:182-200``)
    with no host work between steps."""

    def __init__(self, model: RatchetGPT, cache: KVCache, greedy: bool = False) -> None:
        cache.check_open()
        self.model, self.cache, self.greedy = model, cache, greedy
        self.tokens = torch.zeros((cache.batch, 1), dtype=torch.long, device=cache.device)
        # warm-up step: allocates the cache buffers, and its token is overwritten by the first
        # replay's. In an 8-bit cache that token could raise a block's scale for good, so the
        # step is warmed up on a cache of its own, of one position.
        warm = cache
        if isinstance(cache, Int8KVCache):
            reserve_step(model, cache)
            warm = model.new_cache(cache.batch, max_len=1, dtype=torch.int8)
        stream = torch.cuda.Stream(device=cache.device)
        stream.wait_stream(torch.cuda.current_stream(cache.device))
        with torch.cuda.stream(stream), torch.no_grad():
            model.decode_logits(self.tokens, warm)
        torch.cuda.current_stream(cache.device).wait_stream(stream)
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph), torch.no_grad():
            self.logits = model.decode_logits(self.tokens, cache)
            if greedy:
                decode_greedy(self.logits.float(), self.tokens, cache.pos)

    def step(self, tokens: Tensor) -> Tensor:
        """Logits [B, vocab] for `tokens` [B, 1] at the cache position; advances the cache.
        The returned tensor is overwritten by the next step."""
        if self.greedy:
            raise RuntimeError("a greedy decode graph is stepped with next_greedy()")
        self.tokens.copy_(tokens)
        self.graph.replay()
        self.cache.advance(1)
        return self.logits

    def next_greedy(self) -> Tensor:
        """One greedy step: consumes `tokens` [B, 1] (set by the caller before the first
        step, then each step's picks), leaves this step's logits in `logits` and its argmax
        in `tokens`, and advances the cache by one. Returns `tokens`."""
        if not self.greedy:
            raise RuntimeError("next_greedy() needs a graph built with greedy=True")
        self.graph.replay()
        self.cache.length += 1
        return self.tokens


class _TokenSampler:
    """Next-token choice of ``generate`` (``generate.py:180-197``): greedy at temperature 0,
    otherwise temperature-scaled logits restricted to the top-k values (ties at the k-th
    value kept), softmax, and one multinomial draw on the CPU from ``seed``'s generator."""

    def __init__(self, temperature: float, top_k: int | None, seed: int | None) -> None:
        self.temperature = temperature
        self.top_k = top_k
        self.generator = None if seed is None else torch.Generator("cpu").manual_seed(seed)

    def __call__(self, logits: Tensor) -> int:
        if self.temperature == 0.0:
            return int(logits.argmax(dim=-1).item())
        scaled = logits / self.temperature
        if self.top_k is not None:
            floor = scaled.topk(min(self.top_k, scaled.shape[-1]), dim=-1).values[:, -1:]
            scaled = torch.where(scaled < floor, torch.full_like(scaled, float("-inf")), scaled)
        weights = scaled.softmax(dim=-1).cpu()
        return int(torch.multinomial(weights, 1, generator=self.generator).item())


@torch.no_grad()
def generate(
    model: RatchetGPT,
    vocabulary: tuple[str, ...],
    prompt: str,
    *,
    max_new_tokens: int,
    temperature: float = 1.0,
    top_k: int | None = None,
    seed: int | None = None,
    device: str | torch.device | None = None,
    use_graph: bool = False,
    cache_dtype: torch.dtype | None = None,
) -> str:
    """Sample `max_new_tokens` characters continuing `prompt` and return only the new text
    (``generate.py:135-206``: same arguments, validation and sampling). `use_graph` replays
    the decode step as a HIP graph (GPU only); `cache_dtype` is the key/value cache's
    (``RatchetGPT.new_cache``: e.g. torch.bfloat16, or torch.int8 for codes with scales)."""
    if max_new_tokens < 0:
        raise ValueError("max_new_tokens must be non-negative")
    if temperature < 0:
        raise ValueError("temperature must be non-negative")
    index = {character: position for position, character in enumerate(vocabulary)}
    missing = sorted(set(prompt) - index.keys())
    if missing:
        raise ValueError(f"prompt characters not in the model vocabulary: {missing!r}")
    pick = _TokenSampler(temperature, top_k, seed)
    device = device or next(model.parameters()).device
    window = model.config.block_size
    # an empty prompt starts from token 0, so there is always a position to predict from
    history = [index[character] for character in prompt] or [0]
    history = history[-window:]
    cache = model.new_cache(1, dtype=cache_dtype)
    logits = model.prefill(torch.tensor([history], dtype=torch.long, device=device), cache)
    graph: DecodeGraph | None = None
    produced: list[int] = []
    while len(produced) < max_new_tokens:
        produced.append(pick(logits))
        history.append(produced[-1])
        if len(produced) == max_new_tokens:
            break
        if cache.length >= window:
            # positions are absolute: once the window slides the cache cannot follow, so the
            # window is recomputed (the reference's path for every token)
            recent = torch.tensor([history[-window:]], dtype=torch.long, device=device)
            logits = model(recent)[0][:, -1]
            continue
        token = torch.tensor([[produced[-1]]], dtype=torch.long, device=device)
        if use_graph and graph is None:
            graph = DecodeGraph(model, cache)
        logits = graph.step(token) if graph is not None else model.decode_step(token, cache)
    return "".join(vocabulary[token] for token in produced)
