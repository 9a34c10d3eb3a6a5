"""A decode loop with Hugging Face's ``generate()`` arguments over the int8
Llama/Qwen2 decoder — the counterpart of python/grilly/infer/generation.py:103-206
for batch 1 (the decoder here is the batch-1 decode step of the int8 full-step
configuration).

The loop is built B200-first: ONE captured CUDA graph holds the whole step —
embedding of the token the sampler left on the device, the 24 layers, the head,
the sampler — and the sampler writes its token where the next step's embedding
reads it and appends it to a device history. The host only replays; it reads
back a token per step when there is an end-of-sequence id to stop at (as the
reference reads back only the sampled ids, generation.py:173), and nothing at
all until the end otherwise. The prompt but for its last token goes through
``LlamaDecoder.prefill`` (all rows at once, causal attention over the cache);
the last token is the first step's input.
"""
from __future__ import annotations

from dataclasses import dataclass, fields, replace

import numpy as np

from .. import _C
from .paged import PagedKvCache, PagedStep
from .sampling import Generator, Sampler, _default_generator, sample_rows

__all__ = ["GenerationConfig", "generate", "generate_batch"]


@dataclass
class GenerationConfig:
    """The ``transformers.GenerationConfig`` fields the loop uses, with their defaults (generation.py:66-86)."""
    max_length: int = 20
    max_new_tokens: int | None = None
    do_sample: bool = False
    temperature: float = 1.0
    top_k: int | None = 50
    top_p: float | None = 1.0
    repetition_penalty: float = 1.0
    eos_token_id: int | list | None = None
    pad_token_id: int | None = None
    num_beams: int = 1
    use_cache: bool = True


_FIELDS = {f.name for f in fields(GenerationConfig)}


def generate(model, inputs=None, generation_config: GenerationConfig | None = None, *, generator: Generator | None = None,
             graphed: bool = True, **kwargs) -> np.ndarray:
    """``model``: a ``LlamaDecoder`` with an empty cache. ``inputs``: the prompt's token ids, int [1, length] (or a flat
    list). Returns the sequence, prompt first, as int64 [1, length]; a sequence that ended at ``eos_token_id`` stops
    there. Unknown keyword arguments raise, naming them, as the reference does."""
    if inputs is None:
        inputs = kwargs.pop("input_ids", None)
    if inputs is None:
        raise ValueError("generate() needs `inputs` (or `input_ids`): the prompt's token ids")
    ids = np.asarray(inputs)
    if ids.ndim == 1:
        ids = ids[None]
    if ids.ndim != 2 or ids.shape[0] != 1 or ids.shape[1] == 0 or not np.issubdtype(ids.dtype, np.integer):
        raise ValueError(f"`inputs` must be integer (1, length) with length > 0 (this decoder runs batch 1), got {ids.dtype} {ids.shape}")
    config = replace(generation_config or GenerationConfig())
    unused = [k for k in kwargs if k not in _FIELDS]
    if unused:
        raise ValueError(f"The following `model_kwargs` are not used by the model: {unused}")
    for k, v in kwargs.items():
        setattr(config, k, v)
    if config.num_beams != 1:
        raise NotImplementedError("grilly: generate() with num_beams > 1 (beam search) is not implemented yet")
    if not config.use_cache:
        raise NotImplementedError("grilly: generate(use_cache=False) is not implemented yet")
    prompt = ids.shape[1]
    total = prompt + config.max_new_tokens if config.max_new_tokens is not None else config.max_length
    steps = total - prompt
    if steps <= 0:
        return ids.astype(np.int64)
    cfg = model.cfg
    if total > cfg.max_cache_len + 1:
        raise RuntimeError(f"the cache holds {cfg.max_cache_len} positions; prompt + new tokens = {total}")
    eos = config.eos_token_id
    eos = set() if eos is None else {int(eos)} if isinstance(eos, (int, np.integer)) else {int(e) for e in eos}

    sampler = Sampler(1, cfg.vocab_size, do_sample=config.do_sample, temperature=config.temperature, top_k=config.top_k,
                      top_p=config.top_p, repetition_penalty=config.repetition_penalty, history_capacity=total,
                      draws=max(steps, 1), generator=generator)
    token = _C.Tensor.from_numpy(ids[0, :1].astype(np.int32), persistent=True)  # the step's input; the sampler's output

    def step():
        logits, _ = model.step(token, want_argmax=False)
        sampler.sample(logits, out=token)  # chooses, writes the next input, appends to the device history

    import grilly2_b200 as g
    run = g.graphed(step) if graphed else step
    if prompt > 1:  # the prompt but for its last token: one pass over all its rows
        model.prefill(_C.Tensor.from_numpy(ids[0, :-1].astype(np.int32)))
        token.copy_(_C.Tensor.from_numpy(ids[0, -1:].astype(np.int32)))
    sampler.set_history(ids)
    done = 0
    for _ in range(steps):
        run()
        done += 1
        if eos and int(token.numpy()[0]) in eos:  # the one value read back per step
            break
    out = sampler.history.numpy()[0, :prompt + done]
    return out[None].astype(np.int64)


def _per_request(name: str, value, n: int, off, dtype):
    """A setting for every request: one value for all (None: ``off``), or a sequence of n."""
    values = list(value) if isinstance(value, (list, tuple, np.ndarray)) else [value] * n
    if len(values) != n:
        raise ValueError(f"`{name}` must be one value or one per prompt ({n}), got {len(values)}")
    return np.array([off if v is None else v for v in values], dtype=dtype)


def generate_batch(model, prompts, generation_config: GenerationConfig | None = None, *, min_p=0.0, block_size: int = 64, blocks: int | None = None,
                   generator: Generator | None = None, graphed: bool = True, **kwargs) -> list:
    """``generate()`` for several prompts at once over a paged int8 cache: the prompts run as one ragged step, then every
    step decodes one token of each request still running; the step, block tables and sampler included, is one captured
    graph. ``do_sample``, ``temperature``, ``top_k``, ``top_p`` and ``min_p`` may be sequences with a setting for each prompt. A request
    that ends at ``eos_token_id`` gives its blocks back. ``blocks``: the pool's size (the default holds all requests to the end); a
    pool that runs out raises. Returns a list of int64 arrays, prompt first. No counterpart in the reference (batch 1)."""
    rows = [np.asarray(p).reshape(-1) for p in prompts]
    n = len(rows)
    if n == 0 or any(r.size == 0 or not np.issubdtype(r.dtype, np.integer) for r in rows):
        raise ValueError("`prompts` must be non-empty sequences of integer token ids")
    if any(int(r.max()) > 0x7FFFFFFF or int(r.min()) < -0x80000000 for r in rows):
        raise ValueError("`prompts` holds a token id that 32 bits do not hold")
    config = replace(generation_config or GenerationConfig())
    unused = [k for k in kwargs if k not in _FIELDS]
    if unused:
        raise ValueError(f"The following `model_kwargs` are not used by the model: {unused}")
    for k, v in kwargs.items():
        setattr(config, k, v)
    if config.num_beams != 1:
        raise NotImplementedError("grilly: generate_batch() with num_beams > 1 (beam search) is not implemented yet")
    if not config.use_cache:
        raise NotImplementedError("grilly: generate_batch(use_cache=False) is not implemented yet")
    if config.repetition_penalty not in (None, 1.0):
        raise NotImplementedError("grilly: generate_batch() with a repetition penalty is not implemented yet")
    cfg = model.cfg
    new = [(config.max_new_tokens if config.max_new_tokens is not None else config.max_length - r.size) for r in rows]
    new = [max(v, 0) for v in new]
    steps = max(new)
    if steps == 0:
        return [r.astype(np.int64) for r in rows]
    held = [r.size + v - 1 if v else 0 for r, v in zip(rows, new)]  # cached positions: the last token never is, nor what asks for no token
    if max(held) > cfg.max_cache_len:
        raise RuntimeError(f"a request may hold {cfg.max_cache_len} cached positions; prompt + new tokens = {max(held) + 1}")
    sampled = _per_request("do_sample", config.do_sample, n, False, bool)
    heat = _per_request("temperature", config.temperature, n, 1.0, np.float32)
    if (sampled & ~(heat > 0)).any():
        raise ValueError("`temperature` has to be a strictly positive float, otherwise your next token scores will be invalid. If you're "
                         "looking for greedy decoding strategies, set `do_sample=False`.")
    T = _C.Tensor.from_numpy
    settings = {"temperature": T(np.where(sampled, heat, 0.0).astype(np.float32)),
                "top_k": T(_per_request("top_k", config.top_k, n, 0, np.int32)), "top_p": T(_per_request("top_p", config.top_p, n, 1.0, np.float32)),
                "min_p": T(_per_request("min_p", min_p, n, 0.0, np.float32))}
    eos = config.eos_token_id
    eos = set() if eos is None else {int(eos)} if isinstance(eos, (int, np.integer)) else {int(e) for e in eos}
    if blocks is None:
        blocks = sum(-(-h // block_size) for h in held)
    cache = PagedKvCache.for_model(cfg, seqs=n, blocks=blocks, block_size=block_size)
    uniforms = T((generator or _default_generator).uniform((steps, n)))
    draws, chosen = T(np.zeros(1, dtype=np.int32)), _C.Tensor.empty((n,), "int32")
    first = [r if v else r[:0] for r, v in zip(rows, new)]  # what runs as the prompts' step
    counts, tokens = T(np.array([r.size for r in first], dtype=np.int32)), T(np.concatenate(first).astype(np.int32))

    def run(tokens, counts, step, max_count):
        cache.plan(counts, step)
        sample_rows(model.step_paged(tokens, cache, step, max_count=max_count), uniforms, draws=draws, tokens=chosen, **settings)

    prompt_step = PagedStep(cache, tokens.numel())
    run(tokens, counts, prompt_step, max(r.size for r in first))
    if prompt_step.shortfall():
        raise RuntimeError(f"the pool of {blocks} blocks cannot hold the prompts: {prompt_step.shortfall()} more are needed")
    step = PagedStep(cache, n)
    tokens, counts = _C.Tensor.empty((n,), "int32"), _C.Tensor.empty((n,), "int32")  # the decode step's inputs

    def decode():
        run(tokens, counts, step, 1)

    import grilly2_b200 as g
    decode = g.graphed(decode) if graphed else decode
    out, running = [list(map(int, r)) for r in rows], [v > 0 for v in new]
    gone = [False] * n
    while True:
        for b, t in enumerate(chosen.numpy()):
            if running[b]:
                if t < 0:
                    raise RuntimeError(f"no token can be drawn for request {b}: its logits are no numbers")
                out[b].append(int(t))
                running[b] = len(out[b]) < rows[b].size + new[b] and int(t) not in eos
        over = [not r and not x for r, x in zip(running, gone)]
        if any(over):
            cache.release(T(np.array(over, dtype=np.int32)))
            gone = [not r for r in running]
        live = [b for b in range(n) if running[b]]
        if not live:
            return [np.array(o, dtype=np.int64) for o in out]
        # a request's row in the step: the running ones in order
        row = np.zeros(n, dtype=np.int32)
        row[:len(live)] = [out[b][-1] for b in live]
        tokens.copy_(T(row))
        counts.copy_(T(np.array(running, dtype=np.int32)))
        decode()
        if step.shortfall():
            raise RuntimeError(f"the pool of {blocks} blocks has run out: {len(live)} requests are running")
