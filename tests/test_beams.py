"""CPU: what BeamSearch does on the host - which stream its library calls go to -
with the library's device calls replaced by recorders and tensors on the host."""
import ctypes
import types

import numpy as np
import pytest

torch = pytest.importorskip("torch")
from torch.overrides import TorchFunctionMode  # noqa: E402

import beams  # noqa: E402
import model_synth as ms  # noqa: E402
import quantr  # noqa: E402

SIDE = 0x5000  # the current stream's handle


class OnHost(TorchFunctionMode):
    """Tensors that are asked for on the GPU are made on the host."""

    def __torch_function__(self, func, types_, args=(), kwargs=None):
        kwargs = dict(kwargs or {})
        if "cuda" in str(kwargs.get("device", "")):
            kwargs["device"] = "cpu"
        if func is torch.Tensor.cuda:
            return args[0]
        return func(*args, **kwargs)


class Recorder:
    """quantr with its device calls recorded: name and stream of each."""

    def __init__(self):
        self.calls = []
        self.refuse = set()  # slots that extend leaves as they are
        rec = self

        class Program:
            def __init__(self, jobs):
                list(jobs)

            def run(self, stream=0):
                rec.calls.append(("program", stream))

            def close(self):
                pass

        self.Program = Program
        self.Kv8Pool = self.Kv8Tables = types.SimpleNamespace(of=lambda *a: a)
        self.Kv8Batch = quantr.Kv8Batch

    def lib(self):
        return types.SimpleNamespace(quantr_gpu_device_ptr=lambda p: p.value)

    def register_weights(self, buf):
        pass

    unregister_weights = register_weights

    def kv8_attend_workspace_bytes(self, *a):
        return 4096

    kv8_pages_workspace_bytes = kv8_attend_workspace_bytes

    def kv8_extend_dev(self, pool, tables, slot, n_new, B, ws, ws_bytes, grown=None, stream=0):
        self.calls.append(("kv8_extend_dev", stream))
        if grown:
            s, g = ((ctypes.c_int * B).from_address(p) for p in (slot, grown))
            for i in range(B):
                g[i] = s[i] not in self.refuse

    def logprobs_dev(self, x, ldl, type_, rows, vocab, token, logprob, entropy, k, top_id, top_logprob, ws, ws_bytes,
                     temperature=1.0, lse=None, stream=0):
        self.calls.append(("logprobs_dev", stream))
        for p, n in ((logprob, rows), (entropy, rows), (top_id, rows * k), (top_logprob, rows * k)):
            if n:
                ctypes.memset(p, 0, 4 * n)

    def __getattr__(self, name):
        if name.endswith("_dev"):
            return lambda *a, stream=0, **kw: self.calls.append((name, stream))
        return getattr(quantr, name)


@pytest.fixture
def host(monkeypatch):
    rec = Recorder()
    monkeypatch.setattr(beams, "qr", rec)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: types.SimpleNamespace(cuda_stream=SIDE))
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: None)
    with OnHost():
        yield rec


def model(embd=8):
    spec = ms.Spec(dim=256, hidden_dim=256, n_layers=2, n_heads=4, n_kv_heads=2, vocab_size=300, seq_len=64, wtype=8,
                   head_type=8, embd_type=embd)
    return ms.build(spec, seed=1)


def test_all_calls_go_to_the_current_stream(host):
    """The layers' torch operations and the library's kernels read each other's
    results, so they belong in one stream: torch's current one."""
    search = beams.BeamSearch(model(), beams=3, max_len=64, page_tokens=32, chunk=16)
    search.run(np.arange(20) % 7, 3)
    search.keep(0)
    names = {n for n, _ in host.calls}
    assert {"program", "kv8_append_dev", "kv8_attend_dev", "kv8_select_dev", "kv8_extend_dev", "kv8_compact_dev",
            "logprobs_dev", "dequantize_rows_dev"} <= names
    assert {n for n, s in host.calls if s != SIDE} == set()
    search.close()


def test_a_beam_that_could_not_grow_is_told(host):
    """Lengths follow what the device did, and a beam that it left as it was
    ends the search with an error instead of wrong positions."""
    search = beams.BeamSearch(model(), beams=3, max_len=64, page_tokens=32, chunk=16)
    search.prefill([1] * 10)
    search.select([0, 0, 0])
    host.refuse = {1}
    with pytest.raises(RuntimeError, match="1"):
        search.step([1, 2, 3])
    assert search.lens == [11, 10, 11]
    search.close()


def test_a_prompt_behind_a_prompt_has_to_fit(host):
    search = beams.BeamSearch(model(), beams=2, max_len=64, page_tokens=32, chunk=16)
    search.prefill([1] * 40)
    done = len(host.calls)
    with pytest.raises(ValueError):
        search.prefill([1] * 25)
    assert search.lens == [40, 0] and len(host.calls) == done
    search.prefill([1] * 24)
    assert search.lens == [64, 0]
    search.close()


@pytest.mark.parametrize("beams_,steps", [(2, 0), (2, -3), (20, 4)])
def test_run_refuses_before_it_begins(host, beams_, steps):
    """No steps, or more beams than tokens to begin with: nothing is launched and
    the cache stays as it is."""
    spec = ms.Spec(dim=256, hidden_dim=256, n_layers=1, n_heads=4, n_kv_heads=2, vocab_size=16, seq_len=64, wtype=8,
                   head_type=8, embd_type=8)
    search = beams.BeamSearch(ms.build(spec, seed=1), beams=beams_, max_len=64, page_tokens=32, chunk=16)
    search.prefill([1] * 10)
    done = len(host.calls)
    with pytest.raises(ValueError):
        search.run([1, 2, 3], steps)
    assert len(host.calls) == done and search.lens[0] == 10
    search.close()
