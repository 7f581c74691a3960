"""Decode and evaluation harness: ``beam_generate``, beam search for a decoder over the paged 8-bit cache of
``asr_amd.decoding``, and the greedy-decode evaluation: the reference's ``evaluate_samples``
(src/train.py:36-82) and the prompt assembly of ``ASRModel.generate`` (src/modeling.py:296-334) on top of this
package's extractor / encoder / projector / splice, plus a word error rate that needs no ``evaluate`` / ``jiwer``.

The decoder itself (an HF causal LM) is outside this path: ``evaluate_samples`` takes any ``model`` with the
reference's ``generate(input_features=..., attention_mask=..., max_new_tokens=..., do_sample=False)`` signature.
WER follows the definition the reference's metric implements (``evaluate.load("wer")`` -> jiwer: words split on
whitespace, (substitutions + deletions + insertions) / reference words, pooled over the corpus).  jiwer is not
installed in this environment, so agreement with it is by definition and known-answer tests only: parity unpinned.
"""
from __future__ import annotations

from typing import Iterable, List, Optional, Sequence, Tuple

import torch


def _edit_distance(ref: Sequence[str], hyp: Sequence[str]) -> int:
    """Word-level Levenshtein distance (unit costs)."""
    prev = list(range(len(hyp) + 1))
    for i, r in enumerate(ref, 1):
        cur = [i] + [0] * len(hyp)
        for j, h in enumerate(hyp, 1):
            cur[j] = min(prev[j] + 1, cur[j - 1] + 1, prev[j - 1] + (r != h))
        prev = cur
    return prev[-1]


def word_error_rate(predictions: Iterable[str], references: Iterable[str]) -> float:
    """Corpus WER = sum of word edit distances / sum of reference lengths (src/train.py:79-80)."""
    predictions, references = list(predictions), list(references)
    if len(predictions) != len(references):
        raise ValueError("predictions and references differ in length")
    errors = total = 0
    for p, r in zip(predictions, references):
        rw, pw = r.split(), p.split()
        errors += _edit_distance(rw, pw)
        total += len(rw)
    if total == 0:
        raise ValueError("references contain no words")
    return errors / total


def build_generate_embeds(prompt_embeds: torch.Tensor, prompt_ids: torch.Tensor, audio_embeds: torch.Tensor,
                          audio_chunk_id: int) -> torch.Tensor:
    """initial_embeds of ``ASRModel.generate`` (src/modeling.py:311-327) through the splice kernel.

    prompt_embeds [1, P, D], prompt_ids [1, P], audio_embeds [B, A, D] -> [B, P-1+A, D].  As in the reference, the
    prompt is spliced with the FIRST sample's audio embeddings and then expanded over the batch (:317-327) -- a
    batch > 1 therefore decodes sample 0 B times there; kept identical here, batch 1 is the only meaningful use."""
    from .splice import splice_audio_embeddings

    if prompt_ids.dim() != 2 or prompt_ids.shape[0] != 1:
        raise ValueError("prompt_ids must be [1, P]")
    try:
        first, _, _ = splice_audio_embeddings(prompt_embeds[:1], audio_embeds[:1].to(prompt_embeds.dtype), prompt_ids, None,
                                              audio_chunk_id)
    except ValueError as e:
        raise ValueError("'<|audio_chunk|>' token not found in instruction.") from e  # :314-315
    return first.expand(audio_embeds.shape[0], -1, -1) if audio_embeds.shape[0] > 1 else first


@torch.no_grad()
def beam_generate(decoder, inputs_embeds: torch.Tensor, *, num_beams: int = 5, max_new_tokens: int = 100,
                  eos_token_id: Optional[int] = None, length_penalty: float = 1.0, prompt_lens: Optional[torch.Tensor] = None,
                  check_every: int = 8) -> Tuple[List[List[int]], torch.Tensor]:
    """Beam search from prompt embeddings, as ``decoder.generate(inputs_embeds=..., num_beams=...)`` of the reference's last
    lines (src/modeling.py:329-334) does it, on the device: the selection, the paged 8-bit cache and its attention are those
    of ``asr_amd.decoding``, and the host is asked only every ``check_every`` steps whether all utterances are done.

    ``inputs_embeds`` [B, P, D] on the GPU (``build_generate_embeds``, ``splice_audio_embeddings``), ``prompt_lens`` int [B] if
    the prompts are right-padded.  ``decoder`` has ``num_layers``, ``kv_heads`` and ``head_dim``, ``embed(tokens [S]) -> [S, D]``,
    and is called as ``decoder(embeds [S, n, D], cache, num_beams) -> logits [S, V]`` of every sequence's last new token; for
    each layer it does ``cache.write(k, v, layer=l)`` and ``cache.attend(q, layer=l, num_beams=num_beams)``, and finds the new
    tokens' positions from ``cache.starts`` on.

    A hypothesis ends with ``eos_token_id`` (which is not returned) when it is among the best ``num_beams`` continuations of
    its utterance; its score is its log-probability over its length (the end counted) to the power ``length_penalty``.  An
    utterance is done when it has ``num_beams`` of them and its best running beam, at its present length, is no better than
    the worst.  Returns the best hypothesis of every utterance and the scores, float32 [B]."""
    from .decoding import PAGE, PagedKVCache, beam_select, reorder_states

    if inputs_embeds.dim() != 3 or inputs_embeds.shape[0] < 1 or inputs_embeds.shape[1] < 1:
        raise ValueError("inputs_embeds must be [B, P, D]")
    if max_new_tokens < 1 or check_every < 1:
        raise ValueError("max_new_tokens and check_every must be positive")
    (B, P, _), K, dev = inputs_embeds.shape, num_beams, inputs_embeds.device
    if prompt_lens is None:
        prompt_lens = torch.full((B,), P, dtype=torch.int32, device=dev)
    elif tuple(prompt_lens.shape) != (B,) or bool(((prompt_lens < 1) | (prompt_lens > P)).any()):
        raise ValueError(f"prompt_lens must be [{B}], from 1 to {P}")
    own = max_new_tokens // PAGE + 2  # pages behind the shared ones that a beam can hold
    cache = PagedKVCache(B * K, P + max_new_tokens, decoder.kv_heads, decoder.head_dim, num_layers=decoder.num_layers,
                         num_pages=B * (-(-P // PAGE) + K * own), device=dev)
    prompts = cache.leaders(K)
    prompts.extend(prompt_lens.to(dev))
    logits = decoder(inputs_embeds, prompts, 1)
    logits = logits.unsqueeze(1).expand(B, K, logits.shape[-1])  # beam 0 alone lives; the others' rows are not looked at
    scores = torch.full((B, K), float("-inf"), device=dev)
    scores[:, 0] = 0
    history = torch.zeros((B, K, max_new_tokens), dtype=torch.int64, device=dev)
    ended = torch.full((B, K), float("-inf"), device=dev)  # hypotheses, best first
    ended_tokens, ended_lens = torch.zeros_like(history), torch.zeros((B, K), dtype=torch.int64, device=dev)
    done = torch.zeros((B, 1), dtype=torch.bool, device=dev)
    row = torch.arange(B, device=dev)[:, None]

    def keep(new, tokens, lens):  # the best K of the old hypotheses and the new ones
        nonlocal ended, ended_tokens, ended_lens
        ended, at = torch.cat([ended, new], 1).sort(dim=1, descending=True, stable=True)
        ended, at = ended[:, :K].contiguous(), at[:, :K]
        ended_tokens = torch.cat([ended_tokens, tokens], 1)[row, at]
        ended_lens = torch.cat([ended_lens, lens], 1).gather(1, at)

    for t in range(max_new_tokens):
        step = beam_select(logits, scores, eos_token_id)
        if eos_token_id is not None:
            new = step.cand_scores[:, :K] / float(t + 1) ** length_penalty
            new = new.masked_fill((step.cand_tokens[:, :K] != eos_token_id) | done, float("-inf"))
            keep(new, history[row, step.cand_parents[:, :K]], torch.full_like(ended_lens, t))
            done = done | ((ended[:, -1:] > float("-inf")) & (step.scores[:, :1] / float(t + 1) ** length_penalty <= ended[:, -1:]))
        history = reorder_states(history, step.parents)
        history[:, :, t] = step.tokens
        scores = step.scores
        if t + 1 == max_new_tokens or (t % check_every == check_every - 1 and bool(done.all())):
            break
        cache.reorder(step.parents)
        cache.extend(1)
        logits = decoder(decoder.embed(step.tokens.view(-1)).unsqueeze(1), cache, K)
    cache.check()
    running = (scores / float(t + 1) ** length_penalty).masked_fill(done, float("-inf"))  # what ran to the end without one
    keep(running, history, torch.full_like(ended_lens, t + 1))
    tokens, lens = ended_tokens[:, 0].cpu(), ended_lens[:, 0].cpu()
    return [tokens[b, :lens[b]].tolist() for b in range(B)], ended[:, 0]


@torch.no_grad()
def evaluate_samples(model, tokenizer, feature_extractor, eval_samples, device=None) -> Tuple[List[str], List[str], float]:
    """Same contract as the reference's ``evaluate_samples`` (src/train.py:36-82): greedy decode of every sample,
    one at a time, returns (predictions, references, wer)."""
    if device is None:
        device = model.device
    predictions, references = [], []
    for sample in eval_samples:
        inputs = feature_extractor(sample["audio"]["array"], sampling_rate=16000, return_tensors="pt",
                                   return_attention_mask=True)
        input_features = inputs.input_features.to(device)
        attention_mask = inputs.attention_mask.to(device) if hasattr(inputs, "attention_mask") else None
        generated_ids = model.generate(input_features=input_features, attention_mask=attention_mask, max_new_tokens=100,
                                       do_sample=False)
        predictions.append(tokenizer.decode(generated_ids[0], skip_special_tokens=True))
        references.append(sample.get("text", sample.get("sentence", "")))
    return predictions, references, word_error_rate(predictions, references)
