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
