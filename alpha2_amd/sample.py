"""Text generation from a trained model (packages/train/src/sample.ts:23-201): for each new token the logits behind the last
blockSize tokens (by a forward pass over them, or from kept keys and values where the model allows it: decode.py), then greedy /
top-k / nucleus / full-softmax selection on the host with the reference's arithmetic (f32 storage, double accumulation, stable
descending sorts) and its use of the seeded rng (one draw per sampled token).  sampleTokensBatch does this for several prompts at
once, one pass of the model for all, their keys and values in pages, the selection on the device."""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Callable, List, Optional, Sequence

import numpy as np

from .autograd import Tape
from .backend import TensorData
from .decode import KeptContext, PagedContext, mayMove
from .model import ModelConfig, gptForward


@dataclass
class SampleConfig:
    """packages/core/src/types.ts:145-158."""
    steps: int = 200
    temperature: float = 0.8
    topk: int = 40
    topp: Optional[float] = 1.0


def _stable_desc(values: np.ndarray) -> np.ndarray:
    """Indices by descending value; equal values keep their index order (Array.prototype.sort is stable)."""
    return np.argsort(-values.astype(np.float64), kind="stable")


def selectToken(lastLogits: np.ndarray, rng, temperature: float, topk: int, topP: float) -> int:
    """sample.ts:85-193 for one position.  `lastLogits` is the f32 row already divided by the temperature (when
    positive); it is modified in place exactly as the reference modifies its copy."""
    V = lastLogits.size
    if temperature <= 0:                                                    # sample.ts:85-99: first maximum wins
        return int(np.argmax(lastLogits))
    if 0 < topk < V:                                                        # sample.ts:102-109: ties with the k-th value stay
        threshold = -np.partition(-lastLogits, topk - 1)[topk - 1]
        lastLogits[lastLogits < threshold] = -np.inf
    if 0 < topP < 1:                                                        # sample.ts:112-163
        maxVal = float(np.max(lastLogits))
        if math.isfinite(maxVal):
            fin = np.isfinite(lastLogits)
            p64 = np.where(fin, np.exp(lastLogits.astype(np.float64) - maxVal), 0.0)
            probs = p64.astype(np.float32)
            active = np.nonzero(fin)[0]
            sumExp = float(np.cumsum(p64[active])[-1]) if active.size else 0.0          # sums the unrounded exponentials
            if sumExp > 0 and active.size > 0:
                active = active[_stable_desc(probs[active])]
                target = sumExp * topP
                keptMass, keepCount = 0.0, 0
                while keepCount < active.size:
                    keptMass += float(probs[active[keepCount]])
                    if keptMass >= target:
                        keepCount += 1
                        break
                    keepCount += 1
                if keepCount <= 0:
                    keepCount = 1
                if keptMass <= 0:
                    keptMass = float(probs[active[0]])
                r = rng.next() * keptMass
                cum, sampled = 0.0, int(active[keepCount - 1])
                for i in range(keepCount):
                    cum += float(probs[active[i]])
                    if r < cum:
                        sampled = int(active[i])
                        break
                return sampled
    maxVal = float(np.max(lastLogits))                                      # sample.ts:166-188
    probs = np.exp(lastLogits.astype(np.float64) - maxVal).astype(np.float32)
    sumExp = float(np.cumsum(probs.astype(np.float64))[-1])                 # sums the f32-rounded values, left to right
    probs = (probs.astype(np.float64) / sumExp).astype(np.float32)
    r = rng.next()
    cum = np.cumsum(probs.astype(np.float64))
    hit = np.nonzero(r < cum)[0]
    return int(hit[0]) if hit.size else 0


def _lastRow(config: ModelConfig, params: dict, backend, context: np.ndarray, releaseTensor: Optional[Callable]) -> np.ndarray:
    """The logits behind the last token of `context`, from a forward pass over all of it (sample.ts:48-80)."""
    V = config.vocabSize
    inputData = TensorData((1, context.size), "i32", context.copy())
    tape = Tape()
    logits = gptForward(config, params, backend, tape, inputData)["logits"]
    row = backend.slice(logits.data, [0, context.size - 1, 0], [1, context.size, V]) if hasattr(backend, "slice") else None
    last = np.asarray(row.data if row is not None else logits.data.data.reshape(-1)[(context.size - 1) * V:], dtype=np.float32).reshape(-1).copy()
    if row is not None and releaseTensor is not None:
        releaseTensor(row)
    tape.clear(releaseTensor)
    if releaseTensor is not None:
        releaseTensor(inputData)
    return last


def sampleTokens(config: ModelConfig, params: dict, backend, rng, promptTokens: Sequence[int], sampleConfig: SampleConfig,
                 releaseTensor: Optional[Callable] = None, flushGpu: Optional[Callable] = None) -> np.ndarray:
    """The token loop of sample() (sample.ts:36-198) without the tokenizer: returns prompt + generated ids.  The parameters keep their values
    meanwhile; releaseTensor and flushGpu may move them."""
    steps, temperature, topk = sampleConfig.steps, sampleConfig.temperature, sampleConfig.topk
    topp = sampleConfig.topp
    topP = min(1.0, max(0.0, topp)) if (topp is not None and math.isfinite(topp)) else 1.0
    prompt = np.asarray(promptTokens, dtype=np.int32)
    maxLen = min(prompt.size + steps, config.blockSize)
    tokens = np.zeros(maxLen, dtype=np.int32)
    tokens[: min(prompt.size, maxLen)] = prompt[:maxLen]                    # Int32Array.set of a longer prompt throws in JS;
    if prompt.size > maxLen:                                                # say so instead of truncating silently
        raise ValueError(f"prompt of {prompt.size} tokens exceeds blockSize {config.blockSize}")
    currentLen = int(prompt.size)
    kept = KeptContext.of(config, params, backend, maxLen) if 0 < currentLen < maxLen else None
    try:
        i = 0
        while i < steps and currentLen < config.blockSize:
            last = _lastRow(config, params, backend, tokens[:currentLen], releaseTensor) if kept is None else kept.lastRow(tokens[:currentLen], releaseTensor)
            if temperature > 0:
                last = (last.astype(np.float64) / temperature).astype(np.float32)
            if flushGpu is not None and (i & 7) == 7:
                flushGpu()
            if kept is not None and (((i & 7) == 7 and mayMove(flushGpu)) or (i == 0 and mayMove(releaseTensor))) and not kept.refresh():
                kept.close()
                kept = None
            nxt = selectToken(last, rng, temperature, topk, topP)
            if currentLen < maxLen:
                tokens[currentLen] = nxt
                currentLen += 1
            i += 1
    finally:
        if kept is not None:
            kept.close()
    return tokens[:currentLen]


def sampleTokensBatch(config: ModelConfig, params: dict, backend, rngs: Sequence, prompts: Sequence[Sequence[int]], sampleConfigs,
                      releaseTensor: Optional[Callable] = None, flushGpu: Optional[Callable] = None) -> List[np.ndarray]:
    """What sampleTokens returns for each prompt with its own rng (and, from a sequence of SampleConfig, its own options), but for roundings: sums are
    taken in other orders, which depend on the sequences that are run together, and the selection on the device takes draws and options in 32
    bits where sampleTokens has 64 (of a full softmax over 50304 tokens a draw falls on the other side of a border about once in two thousand, by
    estimate).  Prompts that share an rng draw from it in turn, token by token.  One forward pass serves a token of every sequence; where model
    or backend do not allow that, the sequences are run one after the other."""
    prompts = [np.asarray(p, dtype=np.int32).reshape(-1) for p in prompts]
    configs = [sampleConfigs] * len(prompts) if isinstance(sampleConfigs, SampleConfig) else list(sampleConfigs)
    if len(rngs) != len(prompts) or len(configs) != len(prompts):
        raise ValueError(f"{len(prompts)} prompts, {len(rngs)} rngs, {len(configs)} options")
    for p in prompts:
        if not 0 < p.size <= config.blockSize:
            raise ValueError(f"prompt of {p.size} tokens, where 1 to blockSize {config.blockSize} are taken")
        if p.min() < 0 or p.max() >= config.vocabSize:
            raise ValueError(f"prompt with tokens outside 0 .. {config.vocabSize - 1}")
    if any(c.steps < 0 for c in configs):
        raise ValueError(f"steps {[c.steps for c in configs]}, where 0 and more are taken")
    wanted = [min(p.size + c.steps, config.blockSize) for p, c in zip(prompts, configs)]
    run = [i for i in range(len(prompts)) if wanted[i] > prompts[i].size]
    kept = PagedContext.of(config, params, backend, [wanted[i] for i in run]) if run else None
    if kept is None:
        return [sampleTokens(config, params, backend, r, p, c, releaseTensor, flushGpu) for r, p, c in zip(rngs, prompts, configs)]
    tokens = [np.concatenate([p, np.zeros(n - p.size, np.int32)]) for p, n in zip(prompts, wanted)]
    at = [int(p.size) for p in prompts]                                     # tokens known on the host
    # What selectToken makes of the options, in 32 bits: none is rounded to a number that means something else (a temperature of 0, a
    # nucleus of nothing or of all, a top_k modulo 2^32).
    least, most, below_one = 2.0 ** -126, 2.0 ** 127, 1 - 2.0 ** -24
    warmth = [1.0 if math.isnan(c.temperature) else min(max(c.temperature, least), most) if c.temperature > 0 else 0.0 for c in configs]
    topk = [min(max(c.topk, 0), config.vocabSize) for c in configs]
    topp = [min(max(c.topp, least), below_one) if c.topp is not None and 0 < c.topp < 1 else 1.0 for c in configs]
    options, chosen = {}, []

    def choose(logits: TensorData, seqs: tuple) -> TensorData:
        if seqs not in options:
            options.clear()
            options[seqs] = [TensorData((len(seqs),), dtype, np.array(list(values))) for dtype, values in (
                ("f32", (warmth[i] for i in seqs)), ("i32", (topk[i] for i in seqs)), ("f32", (topp[i] for i in seqs)))]
        # (a draw that f32 would round to 1 stays below it)
        draws = np.array([rngs[i].next() if warmth[i] > 0 else 0.0 for i in seqs]).astype(np.float32)
        r = backend.sampleRows(logits, TensorData((len(seqs),), "f32", np.minimum(draws, np.float32(below_one))), *options[seqs])
        if releaseTensor is not None:
            releaseTensor(logits)
        chosen.append((seqs, r["tokens"]))
        return r["tokens"]

    def settle():
        for seqs, t in chosen:
            for i, token in zip(seqs, t.data):
                tokens[i][at[i]] = token
                at[i] += 1
        chosen.clear()

    try:
        # the prompts, as many rows at a time as the memory for activations is meant for: a long one over several passes
        done = [0] * len(run)
        while any(done[j] < prompts[i].size for j, i in enumerate(run)):
            room, part = kept.MOST_ROWS, []
            for j, i in enumerate(run):
                n = min(room, int(prompts[i].size) - done[j])
                if n > 0:
                    part.append((j, prompts[i][done[j]:done[j] + n]))
                    room -= n
            for j, new in part:
                done[j] += new.size
            ready = [k for k, (j, _) in enumerate(part) if done[j] == prompts[run[j]].size]
            logits = kept.forward([j for j, _ in part], [new.size for _, new in part], np.concatenate([new for _, new in part]), ready, releaseTensor)
            if ready:
                choose(logits, tuple(run[part[k][0]] for k in ready))
        step, last, made = 1, None, [1] * len(run)
        while True:
            live = [j for j, i in enumerate(run) if made[j] < wanted[i] - prompts[i].size]
            if not live:
                break
            seqs = tuple(run[j] for j in live)
            if last is None or last[0] != seqs:                             # (the sequences that are left stay in order)
                settle()
                last = (seqs, np.array([tokens[i][at[i] - 1] for i in seqs], np.int32))
            logits = kept.forward(live, [1] * len(live), last[1], range(len(live)), releaseTensor)
            last = (seqs, choose(logits, seqs))
            for j in live:
                made[j] += 1
            if flushGpu is not None and (step & 7) == 7:
                flushGpu()
            step += 1
        settle()
    finally:
        kept.close()
    return tokens


def sample(config: ModelConfig, params: dict, backend, rng, encode: Callable, decode: Callable, prompt: str, sampleConfig: SampleConfig,
           releaseTensor: Optional[Callable] = None, flushGpu: Optional[Callable] = None) -> str:
    """sample.ts:23-201."""
    return decode(sampleTokens(config, params, backend, rng, encode(prompt), sampleConfig, releaseTensor, flushGpu))
