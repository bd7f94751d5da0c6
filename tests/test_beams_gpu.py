"""GPU: beam search over the 8-bit paged cache, all its operators together."""
import numpy as np
import pytest

import model_synth as ms

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

Q8_0, Q4_K, Q6_K = 8, 12, 14


def small(heads=8, kv=2, hd=0, layers=3, vocab=600):
    spec = ms.Spec(dim=256, hidden_dim=512, n_layers=layers, n_heads=heads, n_kv_heads=kv, vocab_size=vocab, seq_len=192,
                   wtype=Q8_0, head_type=Q8_0, embd_type=Q8_0, head_dim=hd)
    return ms.build(spec, seed=3)


def test_layers_against_attention_in_torch(qr_gpu):
    """The logits of a prompt and of forked steps are those of the same layers
    with plain attention over the cache's own values."""
    import beams

    class Plain(beams.BeamSearch):
        def attend(self, b, batch, layer):
            s, n, B = self.spec, batch.max_rows, batch.B
            table, lens, _ = self.state[0]
            P, G = self.k.shape[3], s.n_heads // s.n_kv_heads
            for q in range(B):
                ln = int(lens[q])
                pages = table[q, :-(-ln // P)].long()
                k, v = (c[pages, layer].float() * z[pages, layer][:, :, None, None] for c, z in
                        ((self.k, self.ks), (self.v, self.vs)))
                k, v = (x.transpose(0, 1).reshape(s.n_kv_heads, -1, s.hd)[:, :ln].repeat_interleave(G, 0) for x in (k, v))
                x = b["qkv"][q * n:(q + 1) * n, :s.q_dim].view(n, s.n_heads, s.hd).transpose(0, 1)
                sc = x @ k.transpose(1, 2) * s.hd ** -0.5
                t, pos = torch.arange(ln, device="cuda"), torch.arange(ln - n, ln, device="cuda")
                sc = sc.masked_fill(t > pos[:, None], float("-inf"))
                b["att"][q * n:(q + 1) * n] = (torch.softmax(sc, 2) @ v).transpose(0, 1).reshape(n, s.q_dim)

    logits = []
    for cls in (beams.BeamSearch, Plain):
        search = cls(small(), beams=3, max_len=192, page_tokens=32, chunk=48)
        got, scores = search.prefill(ms.prompt(search.spec, 100)[0])
        search.select([0, 0, 0])
        steps = [search.step([5, 9, 400]).clone(), search.step([7, 7, 7]).clone()]
        logits.append([got.clone(), scores] + steps)
        assert qr_gpu.device_status() == 0
        search.close()
    # An activation that differs in its last bits may round to another 8-bit
    # code of the next layer's input or of the cache: 2^-7 of a block's largest.
    for a, b in zip(*logits):
        assert float((a - b).abs().max()) <= 2.0 ** -7 * max(1.0, float(b.abs().max()))
        assert float((a - b).norm() / b.norm()) <= 2.0 ** -8


def test_beams_are_their_own_sequences(qr_gpu):
    """Each beam found, decoded again alone from a prompt of its own, scores the
    same; scores fall; all pages come back."""
    import beams
    model = small(heads=4, kv=4, hd=48)
    search = beams.BeamSearch(model, beams=5, max_len=160, page_tokens=32, chunk=32)
    prompt = ms.prompt(model.spec, 70)[0]
    tokens, scores = search.run(prompt, 12)
    assert tokens.shape == (5, 12) and len({tuple(t) for t in tokens}) == 5
    assert np.all(np.diff(scores) <= 0)
    for t, want in zip(tokens, scores):
        search.select([-1] * 5)
        logits, _ = search.prefill(prompt)
        total = 0.0
        for i, tok in enumerate(t):
            got = search.score(logits, 1, 1, torch.tensor([int(tok)], dtype=torch.int32, device="cuda"))
            total += float(got["logprob"][0])
            if i + 1 < len(t):
                # beam 0 alone writes; the others hold nothing
                pos = torch.tensor([search.lens[0]], device="cuda")
                search.extend([0], 1)
                logits = search.forward(torch.tensor([int(tok)], device="cuda"), pos, qr_gpu.Kv8Batch(None, None, 1, 1), 1)
        assert abs(total - want) <= 12 * 2.0 ** -7
    refs = search.state[0][2]
    assert search.keep(0) == -(-(70 + 11) // 32)
    refs = search.state[0][2]
    assert refs[:3].tolist() == [1, 1, 1] and int(refs.sum()) == 3
    search.select([-1] * 5)
    torch.cuda.synchronize()
    assert int(search.state[0][2].abs().sum()) == 0
    assert qr_gpu.device_status() == 0
    search.close()


def test_prefill_chunks_agree(qr_gpu):
    """Chunk sizes that end inside pages change a prompt's scores by no more
    than the cache's rounding: a page's scale may be the largest value's of the
    page or up to twice that."""
    import beams
    model = small()
    got = []
    for chunk in (16, 50, 64):
        search = beams.BeamSearch(model, beams=2, max_len=192, page_tokens=64, chunk=chunk)
        got.append(search.prefill(ms.prompt(model.spec, 130)[0])[1])
        search.close()
    for g in got[1:]:
        assert float((g - got[0]).abs().mean()) <= 0.05
    assert qr_gpu.device_status() == 0


def test_refusals(qr_gpu):
    import beams
    moe = ms.Spec(dim=256, hidden_dim=256, n_layers=1, n_heads=4, n_kv_heads=4, vocab_size=300, seq_len=64, expert_count=4,
                  expert_used_count=2)
    with pytest.raises(ValueError):
        beams.BeamSearch(ms.build(moe), 2, 64)
    model = small()
    with pytest.raises(ValueError):
        beams.BeamSearch(model, 65, 64)
    search = beams.BeamSearch(model, 2, 64)
    with pytest.raises(ValueError):
        search.prefill([])
    with pytest.raises(ValueError):
        search.prefill([1] * 65)
    search.prefill([1] * 64)
    search.select([0, 0])
    with pytest.raises(ValueError):
        search.step([1, 2])
    search.close()
