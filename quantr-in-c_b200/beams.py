"""Beam search on the device over an 8-bit paged KV cache.

Several continuations of one prompt, decoded together: the prompt is written
once and its pages shared (quantr_kv8_select_dev), a continuation gets pages of
its own where it writes (quantr_kv8_extend_dev), attention reads them all in one
call (quantr_kv8_attend_dev), and the next tokens are scored with their
alternatives (quantr_logprobs_dev).  The linear layers are GEMV programs; the
small elementwise steps between them (norms, RoPE, SwiGLU) are torch operations.
All of it runs on torch's current stream.

The reference has neither a batch nor beams (its loop is one greedy sequence,
src/main.c:305-317); the layer is its forward_runtime (src/runtime.c:94-289),
dense FFN only.

    search = BeamSearch(model, beams=4, max_len=1024)
    tokens, scores = search.run(prompt, steps=32)     # best first

    python quantr-in-c_b200/beams.py                  # a small random model
"""
import ctypes

import numpy as np
import torch

import quantr as qr

F32 = qr.F32


def stream():
    """The stream that the torch operations between the library's calls run on."""
    return torch.cuda.current_stream().cuda_stream


class BeamSearch:
    def __init__(self, model, beams, max_len, page_tokens=64, chunk=64, window=0):
        s = model.spec
        if s.expert_count:
            raise ValueError("BeamSearch runs dense models")
        if s.hd % 16 or s.hd > 128:
            raise ValueError("the 8-bit cache takes head dims that are multiples of 16 up to 128")
        if not 1 <= beams <= 64:
            raise ValueError("1 to 64 beams (their alternatives come from one call)")
        self.model, self.spec, self.beams, self.chunk, self.max_len, self.window = model, s, beams, chunk, max_len, window
        L = qr.lib()
        qr.register_weights(model.buf)
        self.addr = lambda name: L.quantr_gpu_device_ptr(ctypes.c_void_p(model.ptr(name)))
        dev = "cuda"

        # The cache: pages for the prompt once and for each beam's own tail.
        P, max_pages = page_tokens, -(-max_len // page_tokens)
        n_pages = (beams + 1) * max_pages
        shape = (n_pages, s.n_layers, s.n_kv_heads, P, s.hd)
        self.k, self.v = (torch.zeros(shape, dtype=torch.int8, device=dev) for _ in range(2))
        self.ks, self.vs = (torch.zeros(shape[:3], device=dev) for _ in range(2))
        self.pool = qr.Kv8Pool.of(self.k, self.v, self.ks, self.vs)
        # Two sets of tables: a step's selection reads one and writes the other.
        self.state = [(torch.full((beams, max_pages), -1, dtype=torch.int32, device=dev),
                       torch.zeros(beams, dtype=torch.int32, device=dev),
                       torch.zeros(n_pages, dtype=torch.int32, device=dev)) for _ in range(2)]
        self.tables = [qr.Kv8Tables.of(*t) for t in self.state]
        self.lens = [0] * beams

        # One query head count, one workspace: chunks of the prompt and steps.
        rows = max(chunk, beams)
        batch = qr.Kv8Batch(None, None, 1, rows)
        self.ws = torch.zeros(max(qr.kv8_attend_workspace_bytes(self.pool, batch, s.n_heads, max_len),
                                  qr.kv8_pages_workspace_bytes(self.pool, self.tables[0])), dtype=torch.uint8, device=dev)
        self.ws_pages = torch.empty_like(self.ws)

        f = lambda name, n: torch.from_numpy(model.array(name).view(np.float32)[:n].copy()).cuda()  # noqa: E731
        self.rms_att = [f(f"rms_att.{i}", s.dim) for i in range(s.n_layers)]
        self.rms_ffn = [f(f"rms_ffn.{i}", s.dim) for i in range(s.n_layers)]
        self.rms_final = f("rms_final", s.dim)
        # The embedding, decoded once.
        self.embd = torch.empty(s.vocab_size, s.dim, device=dev)
        if s.embd_type == F32:
            self.embd.copy_(torch.from_numpy(model.array("token_embd").view(np.float32)).view(s.vocab_size, s.dim))
        else:
            qr.dequantize_rows_dev(self.embd.data_ptr(), s.dim, self.addr("token_embd"), qr.row_bytes(s.embd_type, s.dim),
                                   s.embd_type, s.dim, s.vocab_size, stream=stream())
        # RoPE (src/runtime.c:19-41): the pair at i turns by pos * base^(-i/head_dim).
        i = torch.arange(0, s.q_dim, 2, device=dev, dtype=torch.float64)
        angle = torch.arange(max_len, device=dev)[:, None] * (s.rope_freq_base ** (-i / s.hd))
        self.cos, self.sin = angle.cos().float(), angle.sin().float()
        self.runs = {}

    # ------------------------------------------------------------- the model --

    def _buffers(self, T):
        """Activations and GEMV programs for T tokens."""
        if T in self.runs:
            return self.runs[T]
        s, m = self.spec, self.model
        b = {n: torch.empty(T, w, device="cuda") for n, w in (
            ("x", s.dim), ("xb", s.dim), ("qkv", s.q_dim + 2 * s.kv_dim), ("att", s.q_dim), ("h1", s.hidden_dim),
            ("h3", s.hidden_dim), ("o", s.dim), ("logits", s.vocab_size))}

        def job(name, n, d, x, out, ldo, at=0):
            return (self.addr(name), m.type_of(name), n, d, T, x.data_ptr(), d, out.data_ptr() + 4 * at, ldo)

        ld = s.q_dim + 2 * s.kv_dim
        b["prog"] = []
        for i in range(s.n_layers):
            b["prog"].append([qr.Program(jobs) for jobs in (
                [job(f"wq.{i}", s.q_dim, s.dim, b["xb"], b["qkv"], ld),
                 job(f"wk.{i}", s.kv_dim, s.dim, b["xb"], b["qkv"], ld, s.q_dim),
                 job(f"wv.{i}", s.kv_dim, s.dim, b["xb"], b["qkv"], ld, s.q_dim + s.kv_dim)],
                [job(f"wo.{i}", s.dim, s.q_dim, b["att"], b["o"], s.dim)],
                [job(f"w1.{i}", s.hidden_dim, s.dim, b["xb"], b["h1"], s.hidden_dim),
                 job(f"w3.{i}", s.hidden_dim, s.dim, b["xb"], b["h3"], s.hidden_dim)],
                [job(f"w2.{i}", s.dim, s.hidden_dim, b["h1"], b["o"], s.dim)])])
        b["head"] = qr.Program([job("wcls", s.vocab_size, s.dim, b["xb"], b["logits"], s.vocab_size)])
        self.runs[T] = b
        return b

    @staticmethod
    def _norm(out, x, w):
        torch.mul(w, x * torch.rsqrt((x * x).mean(1, keepdim=True) + 1e-5), out=out)

    def _rope(self, x, pos):
        n = x.shape[1] // 2
        c, s = self.cos[pos, :n], self.sin[pos, :n]
        a, b = x[:, 0::2].clone(), x[:, 1::2].clone()
        x[:, 0::2] = a * c - b * s
        x[:, 1::2] = a * s + b * c

    def attend(self, b, batch, layer):
        s, ld = self.spec, b["qkv"].shape[1]
        qr.kv8_attend_dev(b["att"].data_ptr(), s.q_dim, b["qkv"].data_ptr(), ld, F32, s.n_heads, self.pool,
                          self.tables[0], batch, layer, s.hd ** -0.5, self.max_len, self.ws.data_ptr(), self.ws.numel(),
                          window=self.window, stream=stream())

    def forward(self, tokens, pos, batch, T):
        """Logits (T x vocab) of the tokens at positions pos, the last rows of
        the batch's sequences.  Tokens past the batch's are padding."""
        s, b, at = self.spec, self._buffers(T), stream()
        ld = b["qkv"].shape[1]
        b["x"].copy_(self.embd[tokens])
        for i in range(s.n_layers):
            qkv, o, h, down = b["prog"][i]
            self._norm(b["xb"], b["x"], self.rms_att[i])
            qkv.run(at)
            self._rope(b["qkv"][:, :s.q_dim], pos)
            self._rope(b["qkv"][:, s.q_dim:s.q_dim + s.kv_dim], pos)
            kv = b["qkv"].data_ptr() + 4 * s.q_dim
            qr.kv8_append_dev(kv, ld, kv + 4 * s.kv_dim, ld, F32, self.pool, self.tables[0], batch, i, stream=at)
            self.attend(b, batch, i)
            o.run(at)
            b["x"] += b["o"]
            self._norm(b["xb"], b["x"], self.rms_ffn[i])
            h.run(at)
            b["h1"].copy_(torch.nn.functional.silu(b["h1"]) * b["h3"])
            down.run(at)
            b["x"] += b["o"]
        self._norm(b["xb"], b["x"], self.rms_final)
        b["head"].run(at)
        return b["logits"]

    # ------------------------------------------------------------- the beams --

    def select(self, pick):
        """Beam i goes on from beam pick[i] (-1: ends, and its pages are free
        unless another beam has them)."""
        f = torch.tensor(pick, dtype=torch.int32, device="cuda")
        qr.kv8_select_dev(self.tables[1], self.tables[0], f.data_ptr(), self.pool, stream=stream())
        self.tables.reverse()
        self.state.reverse()
        self.lens = [self.lens[p] if p >= 0 else 0 for p in pick]

    def extend(self, slots, n):
        """Room for n more tokens of the beams in `slots`.  Waits for the
        device: a beam that it left as it was (its table full, or no page left)
        must not go on."""
        slot = torch.tensor(slots, dtype=torch.int32, device="cuda")
        new = torch.full((len(slots),), n, dtype=torch.int32, device="cuda")
        grown = torch.empty_like(slot)
        qr.kv8_extend_dev(self.pool, self.tables[0], slot.data_ptr(), new.data_ptr(), len(slots),
                          self.ws_pages.data_ptr(), self.ws_pages.numel(), grown=grown.data_ptr(), stream=stream())
        done = grown.tolist()
        for i, ok in zip(slots, done):
            self.lens[i] += n if ok else 0
        if not all(done):
            raise RuntimeError(f"no room for beams {[i for i, ok in zip(slots, done) if not ok]}")

    def score(self, logits, rows, k, token=None, temperature=1.0):
        """The k best alternatives of each row with their log probabilities, the
        entropy, and the given tokens' log probabilities."""
        out = {"logprob": torch.empty(rows, device="cuda"), "entropy": torch.empty(rows, device="cuda"),
               "ids": torch.empty(rows, k, dtype=torch.int32, device="cuda"), "top": torch.empty(rows, k, device="cuda")}
        token = torch.full((rows,), -1, dtype=torch.int32, device="cuda") if token is None else token
        qr.logprobs_dev(logits.data_ptr(), logits.stride(0), F32, rows, self.spec.vocab_size, token.data_ptr(),
                        out["logprob"].data_ptr(), out["entropy"].data_ptr(), k, out["ids"].data_ptr(),
                        out["top"].data_ptr(), None, 0, temperature=temperature, stream=stream())
        return out

    def prefill(self, prompt):
        """Writes the prompt into beam 0, behind what it holds, `chunk` tokens at
        a time; the logits of its last token (1 x vocab) and the log probability
        of each prompt token after the first."""
        prompt = torch.as_tensor(np.asarray(prompt, np.int32), device="cuda")
        T, scores, first = self.chunk, [], self.lens[0]
        if not 0 < prompt.numel() <= self.max_len - first:
            raise ValueError("the prompt has to have a token, and max_len has to hold it")
        for at in range(0, prompt.numel(), T):
            part = prompt[at:at + T]
            n = part.numel()
            self.extend([0], n)
            tokens = torch.zeros(T, dtype=torch.long, device="cuda")
            tokens[:n] = part
            pos = torch.arange(first + at, first + at + T, device="cuda").clamp(max=self.max_len - 1)
            batch = qr.Kv8Batch(None, None, 1, n)
            logits = self.forward(tokens, pos, batch, T)
            follow = torch.full((n,), -1, dtype=torch.int32, device="cuda")
            ahead = prompt[at + 1:at + n + 1]
            follow[:ahead.numel()] = ahead
            scores.append(self.score(logits, n, 0, follow)["logprob"])
        return logits[n - 1:n], torch.cat(scores)[:-1]

    def step(self, tokens):
        """One token for every beam: their logits (beams x vocab)."""
        B = self.beams
        if max(self.lens) >= self.max_len:
            raise ValueError("a beam is max_len tokens long already")
        pos = torch.tensor(self.lens, device="cuda")
        self.extend(list(range(B)), 1)
        return self.forward(torch.as_tensor(tokens, device="cuda").long(), pos, qr.Kv8Batch(None, None, B, 1), B)

    def run(self, prompt, steps):
        """The `beams` best continuations of `steps` tokens: int32[beams, steps]
        and the sums of their log probabilities, best first."""
        B = k = self.beams
        if steps < 1:
            raise ValueError("at least one step")
        if self.spec.vocab_size < B:
            raise ValueError("more beams than tokens")
        self.select([-1] * B)
        logits, _ = self.prefill(prompt)
        first = self.score(logits, 1, k)
        tokens = first["ids"].cpu().numpy().T.astype(np.int32)  # (B, 1)
        scores = first["top"].cpu().numpy()[0].astype(np.float64)
        self.select([0] * B)
        for _ in range(steps - 1):
            got = self.score(self.step(tokens[:, -1]), B, k)
            ids, top = got["ids"].cpu().numpy(), got["top"].cpu().numpy().astype(np.float64)
            total = (scores[:, None] + top).reshape(-1)
            best = np.argsort(-total, kind="stable")[:B]
            pick = best // k
            tokens = np.concatenate([tokens[pick], ids.reshape(-1)[best][:, None]], 1)
            scores = total[best]
            self.select([int(p) for p in pick])
        return tokens, scores

    def keep(self, beam):
        """Ends all beams but one and moves its pages to the front of the pool;
        how many there are."""
        live = torch.empty(1, dtype=torch.int32, device="cuda")
        self.select([beam] + [-1] * (self.beams - 1))
        qr.kv8_compact_dev(self.pool, self.tables[0], None, live.data_ptr(), self.ws_pages.data_ptr(),
                           self.ws_pages.numel(), stream=stream())
        return int(live)

    def close(self):
        torch.cuda.synchronize()
        for b in self.runs.values():
            for layer in b["prog"]:
                for p in layer:
                    p.close()
            b["head"].close()
        self.runs = {}
        qr.unregister_weights(self.model.buf)


def main():
    import model_synth as ms
    spec = ms.Spec(dim=512, hidden_dim=1024, n_layers=4, n_heads=8, n_kv_heads=2, vocab_size=2000, seq_len=256,
                   wtype=qr.Q4_K, head_type=qr.Q6_K, embd_type=qr.Q8_0)
    search = BeamSearch(ms.build(spec, seed=1), beams=4, max_len=256)
    tokens, scores = search.run(ms.prompt(spec, 100)[0], 24)
    for t, sc in zip(tokens, scores):
        print(f"{sc:9.3f}  {' '.join(map(str, t))}")
    print("pages kept:", search.keep(0), "status:", qr.device_status())
    search.close()


if __name__ == "__main__":
    main()
