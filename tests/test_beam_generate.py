"""CPU: the search that ``evaluation.beam_generate`` runs -- which hypotheses end, are kept and win -- against HF ``generate`` with the
same model, a tiny randomly initialised one in float64.  The cache is one that keeps every sequence's embeddings, the selection
is the oracle's; their own tests compare the real ones."""
import pytest
import torch

from oracle import decoding as od

transformers = pytest.importorskip("transformers")


class Sequences:
    """What the search asks of a cache: which tokens a sequence has, by their embeddings."""

    def __init__(self, num_seqs, max_len, kv_heads, head_dim, *, num_layers, num_pages, device):
        self.rows, self.every, self.max_len = [[] for _ in range(num_seqs)], 1, max_len

    def leaders(self, num_beams):
        view = object.__new__(Sequences)
        view.rows, view.every, view.max_len = self.rows, num_beams, self.max_len
        return view

    def extend(self, n):
        slots = range(0, len(self.rows), self.every)
        self.new = dict(zip(slots, n.tolist() if isinstance(n, torch.Tensor) else [n] * len(slots)))
        assert all(len(self.rows[s]) + m <= self.max_len for s, m in self.new.items())

    def reorder(self, parents):
        B, K = parents.shape
        self.rows[:] = [list(self.rows[b * K + p]) for b in range(B) for p in parents[b].tolist()]

    def check(self):
        pass


class Decoder:
    num_layers, kv_heads, head_dim = 2, 2, 64

    def __init__(self, model):
        self.model = model

    def embed(self, tokens):
        return self.model.get_input_embeddings()(tokens)

    def __call__(self, embeds, cache, num_beams):
        out = []
        for x, (s, n) in zip(embeds, cache.new.items()):
            cache.rows[s] += list(x[:n])
            out.append(self.model(inputs_embeds=torch.stack(cache.rows[s])[None]).logits[0, -1])
        return torch.stack(out)


def on_the_cpu(monkeypatch):
    from asr_amd import decoding

    def select(logits, scores, eos):
        B, K = scores.shape
        out = od.select(logits.reshape(B, K, -1).numpy(), scores.numpy(), -1 if eos is None else eos)
        return decoding.BeamStep(*map(torch.from_numpy, out))

    monkeypatch.setattr(decoding, "PagedKVCache", Sequences)
    monkeypatch.setattr(decoding, "beam_select", select)
    monkeypatch.setattr(decoding, "reorder_states", lambda x, parents: x[torch.arange(len(x))[:, None], parents])


def tiny(seed, vocab):
    torch.manual_seed(seed)
    config = transformers.LlamaConfig(vocab_size=vocab, hidden_size=32, intermediate_size=48, num_hidden_layers=2, num_attention_heads=2,
                                      num_key_value_heads=1, max_position_embeddings=64, initializer_range=0.6)
    return transformers.LlamaForCausalLM(config).double().eval()


@pytest.mark.parametrize("K", [1, 2, 3, 5])
@pytest.mark.parametrize("penalty", [0.0, 1.0, 2.0])
@pytest.mark.parametrize("vocab,steps", [(7, 12), (40, 9)])
def test_beam_generate_finds_what_generate_finds(monkeypatch, K, penalty, vocab, steps):
    from asr_amd.evaluation import beam_generate

    on_the_cpu(monkeypatch)
    early = 0
    for seed in range(3):
        model, eos = tiny(seed, vocab), 2
        embeds = torch.randn((3, 5, 32), dtype=torch.float64, generator=torch.Generator().manual_seed(seed))
        tokens, scores = beam_generate(Decoder(model), embeds, num_beams=K, max_new_tokens=steps, eos_token_id=eos, length_penalty=penalty, check_every=1 + seed)
        with torch.no_grad():
            want = model.generate(inputs_embeds=embeds, attention_mask=torch.ones((3, 5), dtype=torch.int64), num_beams=K, max_new_tokens=steps, do_sample=False,
                                  length_penalty=penalty, eos_token_id=eos, pad_token_id=0, bos_token_id=1, early_stopping=False, return_dict_in_generate=True,
                                  output_scores=True)
        for b in range(3):
            row = want.sequences[b].tolist()
            row = row[:row.index(eos)] if eos in row else row
            early += len(row) < steps
            assert tokens[b] == row, (seed, b, tokens[b], row)
            if K > 1:
                assert abs(float(scores[b]) - float(want.sequences_scores[b])) <= 1e-5
    assert early > 0 or vocab > 7  # some end before the last step
