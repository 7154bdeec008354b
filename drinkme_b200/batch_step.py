"""A small serving loop over the packed Linears: up to eight sequences at once,
their keys and values in a paged 4-bit cache (kv4), and penalties, biases and a
grammar's mask on the logits (logits) — the decode_step module's stack, widened
from one sequence with a bf16 cache to a batch.

    st = BatchStack(decode_step.QWEN3["qwen3-8b"], seqs=4, max_len=4096)
    st.prefill([[1, 2, 3], [4, 5], [6], [7, 8]])   # any lengths
    st.capture()
    for _ in range(100):
        st.replay()                                 # st.token: the tokens chosen
    st.check()                                      # raises what the kernels recorded

`prefill` runs a ragged batch of prompts: dense Linears (the packed weights decoded, then
cuBLAS: the modules' arm for many rows), one append and one prompt attention a
layer. `step` is one decode step of every sequence, all of it on the device, so it
is captured in one CUDA graph: the packed GEMV of M rows (radix_ops.gemv_into), kv4.append
(q/k RMSNorm, rotary, the 4-bit rows), kv4.attention, the raw lm_head, and
logits.process before the greedy choice. The reference's counterparts are its engine's
batch loop over transformers' modules and caches (src/drinkme/serving/engines.py,
src/drinkme/serving/kvcache.py, src/drinkme/serving/sampling.py).
"""
from __future__ import annotations

import ctypes as ct

import torch

from . import _lib, decode_step, kv4, logits, radix_ops

EPS = decode_step.EPS


def _option(name: str, what: str, dtype: torch.dtype, dim: int) -> property:
    """A tensor of a row a sequence that the captured step reads in place: another one
    in its place means another graph (replay captures it)."""
    key = "_" + name

    def put(self, t) -> None:
        if t is not None and (t.dtype is not dtype or t.dim() != dim or t.shape[0] != self.seqs
                              or (dim == 2 and t.shape[1] < -(-self.s["vocab"] // 32))
                              or t.device != self.token.device or not t.is_contiguous()):
            raise ValueError(f"batch_step: {name} must be a contiguous {what} tensor on {self.token.device}, "
                             f"not {t.dtype} {list(t.shape)} on {t.device}")
        if getattr(self, "graph", None) is not None and t is not getattr(self, key):
            torch.cuda.synchronize(self.dev)  # a replay may still read the old one
            self.graph = None
        setattr(self, key, t)

    return property(lambda self: getattr(self, key), put, doc=what)


class BatchStack:
    """Static buffers of a decode step of `seqs` sequences (1 .. MC_MAX) over
    the packed weights of a decode_step.DecodeStack; see the module docstring.

    What the requests ask for is neutral until set: fill `allowed`, `repetition`,
    `presence` and `frequency` in place at any time, or assign other tensors or
    None (the next replay then captures the step again)."""

    allowed = _option("allowed", "int32 [seqs, ceil(vocab / 32)]", torch.int32, 2)  # bits as in logits.process
    repetition = _option("repetition", "fp32 [seqs]", torch.float32, 1)
    presence = _option("presence", "fp32 [seqs]", torch.float32, 1)
    frequency = _option("frequency", "fp32 [seqs]", torch.float32, 1)

    def __init__(self, shape: dict, device="cuda", seqs: int = 4, max_len: int = 1024, page: int = 64, seed: int = 0,
                 variants: int = 2, layers: int | None = None):
        if not 1 <= seqs <= radix_ops.MC_MAX:
            raise ValueError(f"batch_step: seqs must be 1 .. {radix_ops.MC_MAX}, not {seqs}")
        self.w = decode_step.DecodeStack(shape, device, max_len=1, seed=seed, variants=variants, layers=layers)
        s, dev = self.w.s, self.w.dev
        self.s, self.dev, self.seqs, self.max_len = s, dev, seqs, max_len
        nh, nkv, hd, H, I = s["heads"], s["kv_heads"], s["head_dim"], s["hidden"], s["inter"]
        cols = -(-max_len // page)
        # page j of sequence b: pages of one sequence lie apart, as an allocator leaves them
        self.table = (torch.arange(cols, device=dev)[None, :] * seqs + torch.arange(seqs, device=dev)[:, None]).to(torch.int32)
        self.caches = [kv4.Cache.empty(cols * seqs, page, nkv, hd, dev) for _ in range(s["layers"])]
        self.cos, self.sin = kv4.rope_tables(hd, max_len, decode_step.ROPE_THETA, device=dev)
        # a step's device state
        self.token = torch.zeros(seqs, dtype=torch.int64, device=dev)
        self.kv_len = torch.zeros(seqs, dtype=torch.int32, device=dev)
        self.batch = kv4.Batch(self.table, torch.arange(seqs + 1, dtype=torch.int32, device=dev), self.kv_len,
                               tokens=seqs, max_q=1)
        self.history = torch.zeros(seqs, max_len + 1, dtype=torch.int32, device=dev)
        self.prompt_len = torch.zeros(seqs, dtype=torch.int32, device=dev)
        self.total_len = torch.zeros(seqs, dtype=torch.int32, device=dev)
        self.last = torch.full((seqs,), max_len, dtype=torch.int64, device=dev)  # the history's last column
        self.rows = [0] * seqs  # each sequence's rows, counted on the host
        self.graph = None
        self.repetition = torch.ones(seqs, device=dev)
        self.presence = torch.zeros(seqs, device=dev)
        self.frequency = torch.zeros(seqs, device=dev)
        self.allowed = torch.full((seqs, -(-s["vocab"] // 32)), -1, dtype=torch.int32, device=dev)
        # static activations
        bf = dict(dtype=torch.bfloat16, device=dev)
        self.h, self.x = torch.empty(seqs, H, **bf), torch.empty(seqs, H, **bf)
        self.qkv = torch.empty(seqs, (nh + 2 * nkv) * hd, **bf)
        self.q, self.attn = torch.empty(seqs, nh, hd, **bf), torch.empty(seqs, nh, hd, **bf)
        self.o, self.dn = torch.empty(seqs, H, **bf), torch.empty(seqs, H, **bf)
        self.gu, self.act = torch.empty(seqs, 2 * I, **bf), torch.empty(seqs, I, **bf)
        self.logits = torch.empty(seqs, s["vocab"], **bf)
        self.batch.reserve(self.caches[0], nh)

    # -- decode ----------------------------------------------------------------
    def _room(self) -> None:
        """Refuses a step that a sequence's allocation has no row for."""
        for b, n in enumerate(self.rows):
            if n >= self.max_len:
                raise ValueError(f"batch_step: sequence {b} holds {n} rows, max_len is {self.max_len}")

    def _count(self) -> None:
        self.rows = [n + 1 for n in self.rows]

    def _norm(self, delta, weight) -> None:
        """h += delta, x = RMSNorm(h) * weight, a row at a time."""
        st = radix_ops._stream(self.dev)
        n = self.s["hidden"]
        for i in range(self.seqs):
            _lib.call("dm_step_add_rmsnorm", self.h[i].data_ptr(), delta[i].data_ptr() if delta is not None else None,
                      weight.data_ptr(), self.x[i].data_ptr(), n, ct.c_float(EPS), st)

    def step(self) -> None:
        """Feeds `token`, leaves the next one there. ValueError, before anything is
        launched, when a sequence holds max_len rows already."""
        self._room()
        self._enqueue()
        self._count()

    def _enqueue(self) -> None:
        """A step's launches. Every tensor is static."""
        s, st = self.s, radix_ops._stream(self.dev)
        nh, nkv, hd = s["heads"], s["kv_heads"], s["head_dim"]
        self.kv_len.add_(1)
        self.h.copy_(self.w.embed.index_select(0, self.token))
        delta = None
        for lay, cache in zip(self.w.layers, self.caches):
            self._norm(delta, lay["ln1"])
            radix_ops.gemv_into(lay["qkv"], self.x, None, self.qkv)
            q, k, v = kv4.split_qkv(self.qkv, nh, nkv, hd)
            kv4.append(cache, self.batch, q, k, v, self.cos, self.sin, q_norm=lay["qn"], k_norm=lay["kn"], eps=EPS,
                       q_out=self.q)
            kv4.attention(cache, self.batch, self.q, out=self.attn)
            radix_ops.gemv_into(lay["o"], self.attn.view(self.seqs, nh * hd), None, self.o)
            self._norm(self.o, lay["ln2"])
            radix_ops.gemv_into(lay["gate_up"], self.x, None, self.gu)
            for i in range(self.seqs):
                _lib.call("dm_step_silu_mul", self.gu[i].data_ptr(), self.act[i].data_ptr(), s["inter"], st)
            radix_ops.gemv_into(lay["down"], self.act, None, self.dn)
            delta = self.dn
        self._norm(delta, self.w.norm)
        _lib.call("dm_gemv_raw", self.w.head.data_ptr(), s["vocab"], s["hidden"], self.x.data_ptr(), _lib.DM_BF16,
                  self.seqs, None, self.logits.data_ptr(), _lib.DM_BF16, st)
        self._choose()

    def _choose(self) -> None:
        """The logits with the requests' penalties and masks, in place; the
        greedy token, which joins the history."""
        logits.process(self.logits, history=self.history, prompt_len=self.prompt_len, total_len=self.total_len,
                       repetition=self.repetition, presence=self.presence, frequency=self.frequency,
                       allowed=self.allowed, out=self.logits)
        torch.argmax(self.logits, -1, out=self.token)
        # the host counts the rows (_room); a length that it did not count stays inside all the same
        at = torch.minimum(self.total_len, self.last)
        self.history.scatter_(1, at[:, None], self.token[:, None].to(torch.int32))
        self.total_len.add_(1)

    def capture(self) -> None:
        """Captures one step (a warm-up step on a side stream first, its state rewound)."""
        self._room()
        state = (self.token, self.kv_len, self.total_len, self.history)
        kept = [t.clone() for t in state]
        side = torch.cuda.Stream(self.dev)
        side.wait_stream(torch.cuda.current_stream(self.dev))
        with torch.cuda.stream(side):
            self._enqueue()
        torch.cuda.current_stream(self.dev).wait_stream(side)
        for t, k in zip(state, kept):
            t.copy_(k)
        torch.cuda.synchronize(self.dev)
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph, stream=side):
            self._enqueue()
        torch.cuda.synchronize(self.dev)

    def replay(self) -> None:
        """`step` by its captured graph, with the same refusal."""
        self._room()
        if self.graph is None:
            self.capture()
        self.graph.replay()
        self._count()

    def check(self) -> None:
        """Raises what the steps' kernels recorded since the last check (a position that the
        page table does not cover, a wait that gave up); synchronises. step and
        replay do not ask."""
        self.batch.check()

    # -- prompts -----------------------------------------------------------------
    def prefill(self, prompts: list[list[int]]) -> None:
        """Starts every sequence over with its prompt (at least one token each, all of them
        in the vocabulary) and chooses its first token."""
        if len(prompts) != self.seqs or any(not p or len(p) >= self.max_len for p in prompts):
            raise ValueError(f"batch_step: {self.seqs} prompts of 1 .. {self.max_len - 1} tokens")
        s, dev = self.s, self.dev
        for b, p in enumerate(prompts):
            if min(p) < 0 or max(p) >= s["vocab"]:
                raise ValueError(f"batch_step: prompt {b} has a token outside the vocabulary of {s['vocab']}")
        nh, nkv, hd, I = s["heads"], s["kv_heads"], s["head_dim"], s["inter"]
        lens = [len(p) for p in prompts]
        batch = kv4.Batch.of(self.table, lens, lens)
        self.history.zero_()
        for b, p in enumerate(prompts):
            self.history[b, : len(p)] = torch.tensor(p, dtype=torch.int32)
        self.kv_len.copy_(batch.kv_len)
        self.prompt_len.copy_(batch.kv_len)
        self.total_len.copy_(batch.kv_len)
        self.rows = lens

        def norm(h, w):
            f = h.float()
            return (f * torch.rsqrt(f.pow(2).mean(-1, keepdim=True) + EPS)).to(torch.bfloat16) * w

        def dense(name, x):
            return torch.nn.functional.linear(x, radix_ops.decode_weight(lay[name]))

        h = self.w.embed.index_select(0, torch.tensor([t for p in prompts for t in p], device=dev))
        for lay, cache in zip(self.w.layers, self.caches):
            q, k, v = kv4.split_qkv(dense("qkv", norm(h, lay["ln1"])), nh, nkv, hd)
            q = kv4.append(cache, batch, q, k, v, self.cos, self.sin, q_norm=lay["qn"], k_norm=lay["kn"], eps=EPS)
            h = h + dense("o", kv4.attention(cache, batch, q).view(-1, nh * hd))
            gu = dense("gate_up", norm(h, lay["ln2"]))
            h = h + dense("down", torch.nn.functional.silu(gu[:, :I]) * gu[:, I:])
        batch.check()
        last = norm(h.index_select(0, batch.q_start[1:].long() - 1), self.w.norm)
        self.logits.copy_(radix_ops.gemv_raw(self.w.head, last, None, torch.bfloat16))
        self._choose()


def main(argv=None) -> int:
    """`python -m drinkme_b200.batch_step`: device time of the graphed step of
    a batch of Qwen3-8B-shaped sequences (synthetic weights) after a prompt."""
    import argparse
    import json

    ap = argparse.ArgumentParser()
    ap.add_argument("--shape", choices=tuple(decode_step.QWEN3), default="qwen3-8b")
    ap.add_argument("--seqs", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=500)
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--max-len", type=int, default=4096)
    ap.add_argument("--layers", type=int, default=None)
    a = ap.parse_args(argv)
    if a.prompt + 3 + a.steps > a.max_len:  # three untimed steps
        ap.error(f"a prompt of {a.prompt} and {3 + a.steps} steps do not fit --max-len {a.max_len}")
    st = BatchStack(decode_step.QWEN3[a.shape], "cuda:0", seqs=a.seqs, max_len=a.max_len, seed=11, layers=a.layers)
    g = torch.Generator().manual_seed(1)
    st.repetition.fill_(1.1)
    st.prefill([torch.randint(st.s["vocab"], (a.prompt,), generator=g).tolist() for _ in range(a.seqs)])
    st.capture()
    for _ in range(3):
        st.replay()
    t0, t1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    t0.record()
    for _ in range(a.steps):
        st.replay()
    t1.record()
    torch.cuda.synchronize()
    st.check()
    ms = t0.elapsed_time(t1) / a.steps
    print(json.dumps({"shape": a.shape, "layers": st.s["layers"], "seqs": a.seqs, "prompt": a.prompt, "steps": a.steps,
                      "ms_per_step": round(ms, 4), "tokens_per_s": round(1e3 * a.seqs / ms, 2),
                      "cache_bytes_per_token_and_layer": st.s["kv_heads"] * (st.s["head_dim"] + 8)}))
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
