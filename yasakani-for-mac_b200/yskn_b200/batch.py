"""A batch of requests that share a prompt prefix, on the stack's attention layers.

The serving loop that the batch operators are made for, each called where a program would
call it. One step of every request that has tokens to run:
  batch_plan        blocks for the new tokens from the pool, their slots and positions
  embedding row -> per layer (residual + norm -> q/k/v operator -> paged_prep (heads into the
  paged cache) -> prefix_attention -> o operator -> residual + norm -> MLP) -> final norm
  head              of each request's last token
  logits_adjust     the requests' penalties, biases and masks, by what each has said so far
  head_select       their next tokens, appended on the device
The shared prefix runs once (fill_prefix, as one request without a prefix); its blocks are
then read by every request and never written again. Weights are the stack's seeded ones
(yskn_b200.stack), every layer a full-attention layer, the cache bf16 in blocks. Everything a
step reads or writes stays on the device and keeps its address, so a decode step (one token
for each request) can be captured as a CUDA graph.

python -m yskn_b200.batch runs 64 requests behind a prefix on four layers and prints the
time of a decode step.
"""
import numpy as np

import yskn_b200 as Y
from yskn_b200 import stack as S

ROT = 64  # rotated channels of a head
THETA = 1e7


class BatchStack(S.Stack):
    """batch requests of up to `capacity` own tokens each, steps of up to max_tokens tokens,
    n_blocks blocks of block_size cache rows shared by the prefix and the requests."""

    def __init__(self, device, layers=4, vocab=S.VOCAB, batch=64, max_tokens=512, capacity=512, n_blocks=1024,
                 block_size=64, bits=8, seed=1):
        super().__init__(device, vocab=vocab, ctx=0, bits=bits, seed=seed, kinds=["attn"] * layers)
        torch = self.torch
        self.batch, self.max_tokens, self.capacity, self.block_size = batch, max_tokens, capacity, block_size
        f32 = lambda *s: torch.zeros(s, dtype=torch.float32, device=device)  # noqa: E731
        i16 = lambda *s: torch.zeros(s, dtype=torch.int16, device=device)  # noqa: E731
        i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device=device)  # noqa: E731
        for L in self.L:  # a block's rows of a head adjacent; seen as [block][row][head][channel]
            L["pages"] = [i16(n_blocks, S.N_KVH, block_size, S.HEAD).transpose(1, 2) for _ in range(2)]
        self.inv_freq = torch.from_numpy((THETA ** (-2.0 * np.arange(ROT // 2) / ROT)).astype(np.float32)).to(device)
        # block pool, the requests' tables and lengths, the shared prefix
        self.pool = torch.arange(n_blocks, dtype=torch.int32, device=device)
        self.free, self.free_out = i32(1).fill_(n_blocks), i32(1)
        self.tables = i32(batch, -(-capacity // block_size))
        self.lens, self.lens_out, self.new = i32(batch), i32(batch), i32(batch)
        self.starts = i32(batch + 1)
        self.prefix_len, self.prefix_blocks = 0, None
        # a request's own tokens (its prompt, then its answers) and how many there are
        self.text, self.said, self.prompt = i32(batch, capacity), i32(batch), i32(batch)
        # controls of the selection, by request; neutral until set
        self.repetition, self.presence, self.frequency = f32(batch) + 1.0, f32(batch), f32(batch)
        self.mask = i32(batch, -(-vocab // 32)).fill_(-1)
        # a step's rows
        T = max_tokens
        self.slots = torch.zeros(T, dtype=torch.int64, device=device)
        self.pos, self.requests = i32(T), i32(T)
        self.tokens = i32(T)
        self.bh, self.bx, self.binv, self.bproj = i16(T, S.HIDDEN), f32(T, S.HIDDEN), f32(T), f32(T, S.HIDDEN)
        self.bq, self.bk, self.bv = f32(T, S.N_QH, 2 * S.HEAD), f32(T, S.N_KVH, S.HEAD), f32(T, S.N_KVH, S.HEAD)
        self.bquery, self.bout = i16(T, S.N_QH, S.HEAD), i16(T, S.N_QH, S.HEAD)
        self.ba_in = f32(T, S.N_QH * S.HEAD)
        self.bg, self.bu, self.bm = f32(T, S.FFN), f32(T, S.FFN), f32(T, S.FFN)
        self.blogits, self.btoken = f32(batch, vocab), i32(batch)
        L = self.L[0]
        sets = [[L["q"], L["k"], L["v"]], [L["o"]], [L["gate"], L["up"]], [L["down"]]]
        n = max([Y.linear_work_bytes(s, T) for s in sets] + [Y.linear_work_bytes([self.head], batch)])
        self.bwork = torch.empty(n, dtype=torch.uint8, device=device)
        n = max(Y.prefix_attention_work_bytes(T, batch, T, S.N_QH, S.N_KVH, S.HEAD),
                Y.prefix_attention_work_bytes(T, 1, T, S.N_QH, S.N_KVH, S.HEAD))
        self.attn_work = torch.empty(n, dtype=torch.uint8, device=device)

    def fill_prefix(self, tokens, stream=None):
        """Runs `tokens` (int32, on the device) once as what every request's text follows. Before any
        request: the pool is as at the start."""
        torch, P = self.torch, tokens.numel()
        if stream is not None:  # torch's operations between the library's calls run on it too
            with torch.cuda.stream(stream):
                return self.fill_prefix(tokens)
        if -(-P // self.block_size) > self.pool.numel():  # the plan would let the rest wait
            raise Y.YsknError(Y.EINVAL, "fill_prefix: more tokens than the pool's blocks hold")
        table = torch.zeros((1, -(-P // self.block_size)), dtype=torch.int32, device=self.dev)
        lens, lens_out, new = (torch.zeros(1, dtype=torch.int32, device=self.dev) for _ in range(3))
        starts = torch.zeros(2, dtype=torch.int32, device=self.dev)
        for at in range(0, P, self.max_tokens):
            n = min(self.max_tokens, P - at)
            new.fill_(n)
            Y.batch_plan(lens, new, table, self.pool, self.free, self.block_size, lens_out, self.free_out, starts,
                         self.slots[:n], self.pos[:n], self.requests[:n])
            self.tokens[:n].copy_(tokens[at:at + n])
            self._layers(n, n, table, lens_out, starts, None, 0)
            lens.copy_(lens_out)
            self.free.copy_(self.free_out)
        self.prefix_len, self.prefix_blocks = P, table[0]

    def say(self, request, tokens):
        """The request's own prompt (a list of token numbers); the next step that gives it
        len(tokens) new tokens runs it."""
        n = len(tokens)
        self.text[request, :n] = self.torch.tensor(tokens, dtype=self.torch.int32, device=self.dev)
        self.said[request] = n
        self.prompt[request] = n

    def step(self, n_tokens, max_new, stream=None):
        """Runs self.new[i] tokens of each request i that said them (a negative number ends the
        request): n_tokens in all at most, max_new for one request at most. A request whose tokens or
        blocks do not fit waits (its length in self.lens stays). Those that ran to the end of what they
        said have their next token appended. Everything runs on `stream` (the current one without it),
        after what the caller has put there."""
        torch, T, W = self.torch, n_tokens, self.capacity
        if stream is not None:
            with torch.cuda.stream(stream):
                return self.step(n_tokens, max_new)
        Y.batch_plan(self.lens, self.new, self.tables, self.pool, self.free, self.block_size, self.lens_out,
                     self.free_out, self.starts, self.slots[:T], self.pos[:T], self.requests[:T], self.prefix_len)
        # token t is its request's text at its position behind the prefix (past the last one: any)
        at = self.requests[:T].clamp(min=0).long() * W + (self.pos[:T] - self.prefix_len).clamp(0, W - 1)
        self.tokens[:T].copy_(self.text.view(-1)[at])
        self._layers(T, max_new, self.tables, self.lens_out, self.starts, self.prefix_blocks, self.prefix_len)
        # each request's last token; a request without one answers with a row that is not used
        last = (self.starts[1:] - 1).clamp(min=0).long()
        Y.linear([self.head], self.bx[last], self.bwork, [self.blogits], inv_rms=self.binv[last])
        Y.logits_adjust(self.blogits, self.blogits, history=self.text, history_lens=self.said,
                        prompt_lens=self.prompt, repetition=self.repetition, presence=self.presence,
                        frequency=self.frequency, mask=self.mask)
        Y.head_select(self.blogits, token=self.btoken)
        own = self.lens_out - self.prefix_len * (self.lens_out > 0)
        spoke = (self.starts[1:] > self.starts[:-1]) & (own == self.said) & (self.said < W)
        place = self.said.clamp(max=W - 1).long().unsqueeze(1)
        self.text.scatter_(1, place, torch.where(spoke, self.btoken, self.text.gather(1, place)[:, 0]).unsqueeze(1))
        self.said.add_(spoke)
        self.lens.copy_(self.lens_out)
        self.free.copy_(self.free_out)

    def _layers(self, T, max_new, tables, lens, starts, prefix_blocks, prefix_len):
        """The first T of self.tokens through every layer, into self.bx and self.binv."""
        h, x, inv, proj = self.bh[:T], self.bx[:T], self.binv[:T], self.bproj[:T]
        q, k, v, query, out = self.bq[:T], self.bk[:T], self.bv[:T], self.bquery[:T], self.bout[:T]
        gate, up, m, a_in = self.bg[:T], self.bu[:T], self.bm[:T], self.ba_in[:T]
        self.embedding.lookup(self.tokens[:T], h)
        before = None
        for L in self.L:
            Y.residual_prepare(h, before, L["in_norm"], S.EPS, x, inv)
            Y.linear([L["q"], L["k"], L["v"]], x, self.bwork, [q, k, v], inv_rms=inv)
            Y.paged_prep(q[:, :, :S.HEAD], k, v, self.slots[:T], self.pos[:T], query, *L["pages"],
                         inv_freq=self.inv_freq, q_norm=L["q_norm"], k_norm=L["k_norm"], eps=S.EPS)
            Y.prefix_attention(query, *L["pages"], tables, lens, starts, max_new, self.attn_work, out,
                               prefix_blocks=prefix_blocks, prefix_len=prefix_len, gate=q[:, :, S.HEAD:])
            Y.widen_bf16(out, a_in)
            Y.linear([L["o"]], a_in, self.bwork, [proj])
            Y.residual_prepare(h, proj, L["post_norm"], S.EPS, x, inv)
            Y.linear([L["gate"], L["up"]], x, self.bwork, [gate, up], inv_rms=inv)
            Y.gated_product(gate, up, m)
            Y.linear([L["down"]], m, self.bwork, [proj])
            before = proj
        Y.residual_prepare(h, before, self.final_norm, S.EPS, x, inv)


def main():
    import torch
    dev = torch.device("cuda:0")
    batch, prefix = 64, 2000
    st = BatchStack(dev, batch=batch)
    gen = torch.Generator(device=dev)
    gen.manual_seed(3)
    stream = torch.cuda.Stream(dev)
    with torch.cuda.stream(stream):
        st.fill_prefix(torch.randint(st.vocab, (prefix,), dtype=torch.int32, device=dev, generator=gen), stream)
        for i in range(batch):
            st.say(i, [(37 * i + 11 * j) % st.vocab for j in range(1 + i % 8)])
        st.presence.fill_(0.5)
        st.new.copy_(st.said)
        st.step(int(st.said.sum()), 8, stream)  # every prompt
        st.new.fill_(1)
        st.step(batch, 1, stream)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            st.step(batch, 1, stream)
        graph.replay()
        steps = 64
        t0, t1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        t0.record()
        for _ in range(steps):
            graph.replay()
        t1.record()
        torch.cuda.synchronize()
    Y.check(Y.status(stream), "batch")
    ms = t0.elapsed_time(t1) / steps
    print("%d requests behind %d shared tokens, %d attention layers: %.3f ms a step, %.0f tokens/s"
          % (batch, prefix, st.layers, ms, batch * 1e3 / ms))
    print("request 0:", st.text[0, :int(st.said[0])].tolist()[:16], "...")


if __name__ == "__main__":
    main()
