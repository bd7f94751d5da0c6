"""GPU: beam search on another stream than the default one."""
import numpy as np
import pytest

import model_synth as ms

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def test_side_stream(qr_gpu):
    """Made and run on a side stream, while the default stream is kept busy: the
    same tokens and scores."""
    import beams
    spec = ms.Spec(dim=256, hidden_dim=512, n_layers=3, n_heads=8, n_kv_heads=2, vocab_size=600, seq_len=192, wtype=8,
                   head_type=8, embd_type=8)
    model = ms.build(spec, seed=3)
    prompt = ms.prompt(spec, 100)[0]
    want = beams.BeamSearch(model, beams=4, max_len=192, page_tokens=32, chunk=48)
    tokens, scores = want.run(prompt, 16)
    want.close()
    busy = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        search = beams.BeamSearch(model, beams=4, max_len=192, page_tokens=32, chunk=48)
        for _ in range(3):
            with torch.cuda.stream(torch.cuda.default_stream()):
                for _ in range(20):
                    busy = (busy @ busy).clamp_(-1, 1)
            got, sc = search.run(prompt, 16)
            assert np.array_equal(got, tokens) and np.array_equal(sc, scores)
        assert search.keep(0) == -(-115 // 32)
    assert qr_gpu.device_status() == 0
    search.close()


def test_a_pool_that_runs_out_ends_the_search(qr_gpu):
    """No page left for some beams: an error, lengths as on the device, and the
    beams that did grow hold their pages."""
    import beams
    spec = ms.Spec(dim=256, hidden_dim=256, n_layers=1, n_heads=4, n_kv_heads=4, vocab_size=300, seq_len=96, wtype=8,
                   head_type=8, embd_type=8)
    search = beams.BeamSearch(ms.build(spec, seed=3), beams=4, max_len=96, page_tokens=32, chunk=32)
    search.prefill(ms.prompt(spec, 64)[0])
    search.select([0, 0, 0, 0])
    refs = search.state[0][2]
    free = (refs == 0).nonzero().flatten().tolist()
    for page in free[2:]:
        refs[page] = 1  # held by somebody else: two pages left for four beams
    with pytest.raises(RuntimeError, match=r"\[2, 3\]"):
        search.step([1, 2, 3, 4])
    assert search.lens == [65, 65, 64, 64] == search.state[0][1].tolist()
    assert qr_gpu.device_status() != 0
    assert qr_gpu.device_status() == 0
    search.close()


def test_a_prompt_in_two_parts(qr_gpu):
    """A second prefill goes on behind the first: the logits of a prompt given
    in two parts are those of the whole.  (Its second part begins a page, so the
    cache holds the same codes: what is left is rounding of the activations to 8
    bits, 2^-7 of a block's largest.)"""
    import beams
    spec = ms.Spec(dim=256, hidden_dim=512, n_layers=2, n_heads=8, n_kv_heads=2, vocab_size=600, seq_len=192, wtype=8,
                   head_type=8, embd_type=8)
    model = ms.build(spec, seed=5)
    prompt = ms.prompt(spec, 96)[0]
    got = []
    for parts in ([prompt], [prompt[:64], prompt[64:]]):
        search = beams.BeamSearch(model, beams=2, max_len=192, page_tokens=32, chunk=32)
        for p in parts:
            logits, scores = search.prefill(p)
        got.append((logits.clone(), scores[-31:].clone()))
        assert search.lens == [96, 0]
        search.close()
    for a, b in zip(*got):
        assert float((a - b).abs().max()) <= 2.0 ** -7 * max(1.0, float(b.abs().max()))
    assert qr_gpu.device_status() == 0
