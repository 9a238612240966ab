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

Where a draft (a small model, n-grams) proposes a tree of tokens for each request, verify runs all of
its nodes in one step in place of step: tree_plan and tree_attention let a node see its own ancestors
only, tree_accept finds the path that is the model's own, cache_compact makes that path's rows
adjacent in every layer and batch_edit gives the other rows' blocks back. fork lets requests
continue others (beams, several answers to one prompt): batch_edit and cache_copy. With logprobs
the log probability of each chosen token, its row's entropy and the likeliest tokens are kept.

python -m yskn_b200.batch runs 64 requests behind a prefix on four layers and prints the
time of a decode step and of a step that verifies eight nodes a request.
"""
import numpy as np

import yskn_b200 as Y
from yskn_b200 import stack as S

ROT = 64  # rotated channels of a head
THETA = 1e7


class BatchStack(S.Stack):
    """batch requests of up to `capacity` own tokens each, steps of up to max_tokens tokens,
    n_blocks blocks of block_size cache rows shared by the prefix and the requests. nodes: of a request's drafted
    tree, at most, its next token among them (0: verify is not used). logprobs: None, or how many of the likeliest
    tokens to keep beside the chosen ones' log probabilities."""

    def __init__(self, device, layers=4, vocab=S.VOCAB, batch=64, max_tokens=512, capacity=512, n_blocks=1024,
                 block_size=64, bits=8, seed=1, nodes=0, logprobs=None):
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
        # all layers' caches; copies of requests
        self.caches = Y.CacheSet([c for L in self.L for c in L["pages"]])
        self.tables_out, self.copies, self.n_copies = i32(batch, self.tables.shape[1]), i32(3, n_blocks), i32(1)
        self.whole = i32(batch).fill_(2 ** 31 - 1)
        # chosen tokens' log probabilities, by request
        self.logprobs = logprobs
        rows = lambda n: (f32(n, 1), f32(n), f32(n, logprobs or 0), i32(n, logprobs or 0))  # noqa: E731
        if logprobs is not None:
            self.logprob, self.entropy, self.top_logprobs, self.top_ids = rows(batch)
        # drafted trees: node j of request i is draft[i][j] behind node draft_parents[i][j]; node 0 its next token
        self.nodes = nodes
        if nodes:
            self.draft_tokens, self.draft_parents = i32(batch, nodes), i32(batch, nodes).fill_(-1)
            self.parents, self.tree, self.tree_pos = i32(T), i32(T, -(-nodes // 32)), i32(T)
            self.path, self.accepted, self.keep, self.next = i32(batch, nodes), i32(batch), i32(batch), i32(batch)
            self.tlogits, self.choice = f32(T, vocab), i32(T)
            self.bwork = torch.empty(max(self.bwork.numel(), Y.linear_work_bytes([self.head], T)), dtype=torch.uint8,
                                     device=device)
            if logprobs is not None:  # by node
                self.node_logprob, self.node_entropy, self.node_top_logprobs, self.node_top_ids = rows(T)

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
        if self.logprobs is not None:
            self._score(self.blogits, self.btoken, self.logprob, self.entropy, self.top_logprobs, self.top_ids)
        own = self.lens_out - self.prefix_len * (self.lens_out > 0)
        spoke = (self.starts[1:] > self.starts[:-1]) & (own == self.said) & (self.said < W)
        place = self.said.clamp(max=W - 1).long().unsqueeze(1)
        self.text.scatter_(1, place, torch.where(spoke, self.btoken, self.text.gather(1, place)[:, 0]).unsqueeze(1))
        self.said.add_(spoke)
        self.lens.copy_(self.lens_out)
        self.free.copy_(self.free_out)

    def _score(self, logits, token, logprob, entropy, top_logprobs, top_ids):
        """The tokens' log probabilities (after penalties, biases and masks) and their rows' likeliest tokens."""
        most = dict(top_logprobs=top_logprobs, top_ids=top_ids) if self.logprobs else {}
        Y.token_logprobs(logits, token.unsqueeze(1), logprob, entropy, **most)

    def draft(self, request, tokens, parents):
        """The request's drafted tree: node j + 1 is tokens[j] behind node parents[j] <= j (node 0 is the request's
        next token, said but not run yet). The next verify that gives it 1 + len(tokens) new tokens runs it."""
        n = len(tokens)
        if (not 0 <= request < self.batch or n >= self.nodes or len(parents) != n or
                any(not 0 <= p <= j for j, p in enumerate(parents))):
            raise Y.YsknError(Y.EINVAL, "draft: a request of the batch, %d nodes at most, each behind an earlier one"
                              % max(self.nodes - 1, 0))
        dev, t = self.dev, self.torch
        self.draft_tokens[request, 1:n + 1] = t.tensor(tokens, dtype=t.int32, device=dev)
        self.draft_parents[request, 1:n + 1] = t.tensor(parents, dtype=t.int32, device=dev)

    def verify(self, n_tokens, stream=None):
        """Runs the trees of the requests that have drafted some: self.new[i] nodes of request i (0: none; 1: its next
        token alone), n_tokens in all at most. The tokens of each accepted path and the model's choice behind it are
        appended; the cache keeps the path's rows. A request that has not run all it said but the last token waits, as
        one whose rows do not fit does: a prompt that step has not run to its end, a fork whose copy did not fit. Paths
        end where the text does, with its last token run and nothing behind it.
        Choices are those that steps with the request's controls as they are would make: a node's penalties count what
        its ancestors and itself say, and the request's mask holds for every node."""
        torch, T, W = self.torch, n_tokens, self.capacity
        if not self.nodes or not 0 < T <= self.max_tokens:
            raise Y.YsknError(Y.EINVAL, "verify: a loop made for trees, and 1..%d tokens" % self.max_tokens)
        if stream is not None:
            with torch.cuda.stream(stream):
                return self.verify(n_tokens)
        own = self.lens - self.prefix_len * (self.lens > 0)
        new = torch.where((own == self.said - 1) | (self.new < 0), self.new, 0)
        Y.batch_plan(self.lens, new, self.tables, self.pool, self.free, self.block_size, self.lens_out,
                     self.free_out, self.starts, self.slots[:T], self.pos[:T], self.requests[:T], self.prefix_len)
        request = self.requests[:T].clamp(min=0).long()
        node = (torch.arange(T, device=self.dev) - self.starts[request]).clamp(0, self.nodes - 1)
        said = self.text.gather(1, (self.said - 1).clamp(min=0).long().unsqueeze(1))[:, 0]
        self.tokens[:T].copy_(torch.where(node > 0, self.draft_tokens[request, node], said[request]))
        self.parents[:T].copy_(self.draft_parents[request, node])
        Y.tree_plan(self.parents[:T], self.requests[:T], self.starts, self.lens_out, self.tree[:T], self.tree_pos[:T])
        self._layers(T, self.nodes, self.tables, self.lens_out, self.starts, self.prefix_blocks, self.prefix_len,
                     self.tree_pos[:T], self.tree[:T])
        logits, choice = self.tlogits[:T], self.choice[:T]
        Y.linear([self.head], self.bx[:T], self.bwork, [logits], inv_rms=self.binv[:T])
        self._adjust_nodes(logits, request)
        Y.head_select(logits, token=choice)
        if self.logprobs is not None:
            self._score(logits, choice, self.node_logprob[:T], self.node_entropy[:T], self.node_top_logprobs[:T],
                        self.node_top_ids[:T])
        # (a node behind the text's last place follows none, so that no path has it)
        fits = torch.where(self.tree_pos[:T] - self.prefix_len < W, self.parents[:T], -1)
        Y.tree_accept(self.tokens[:T], fits, choice, self.starts, self.lens_out, self.path, self.accepted,
                      self.keep, self.next)
        Y.cache_compact(self.caches, self.tables, self.lens_out, self.starts, self.path, self.prefix_len)
        Y.batch_edit(self.lens_out, self.keep, self.tables, self.pool, self.free_out, self.block_size, self.lens,
                     self.free, prefix_len=self.prefix_len)
        # the path's tokens behind node 0, then the choice after its last node
        at = self.starts[:-1, None].long() + self.path[:, 1:].clamp(min=0)
        took = torch.cat([self.tokens[at.clamp(max=T - 1)], self.next.unsqueeze(1)], 1)
        count = self.accepted.long().unsqueeze(1)
        col = torch.arange(W, device=self.dev).unsqueeze(0) - self.said.unsqueeze(1)
        new = torch.where(col == count - 1, self.next.unsqueeze(1), took.gather(1, col.clamp(0, self.nodes - 1)))
        self.text.copy_(torch.where((col >= 0) & (col < count), new, self.text))
        self.said.copy_((self.said + self.accepted).clamp(max=W))

    def _adjust_nodes(self, logits, request):
        """The controls of each node's request on its logits: its history is the request's text, then the tokens from
        node 1 on of the path that leads to it, its own the last."""
        torch, T, N = self.torch, logits.shape[0], self.nodes
        first = self.starts[:-1].long()[request].clamp(max=T - 1)
        node = torch.arange(N, device=self.dev).unsqueeze(0)
        at = (first.unsqueeze(1) + node).clamp(max=T - 1)  # of each node of the same tree
        depth = self.tree_pos[:T] - self.tree_pos[first]  # of each token; what follows no one here has 0
        sees = (self.tree[:T].gather(1, (node >> 5).expand(T, N)) >> (node & 31)) & 1 == 1
        said, end = self.said[request], self.capacity + N  # a history's last place: for what it does not hold
        history = torch.cat([self.text, self.text.new_zeros(self.batch, N + 1)], 1)[request]
        place = torch.where(sees & (depth[at] > 0), said.unsqueeze(1) - 1 + depth[at], end)
        history.scatter_(1, place.clamp(0, end).long(), self.tokens[at])
        Y.logits_adjust(logits, logits, history=history[:, :end], history_lens=said + depth.clamp(min=0),
                        prompt_lens=self.prompt[request], repetition=self.repetition[request],
                        presence=self.presence[request], frequency=self.frequency[request], mask=self.mask[request])

    def fork(self, source, stream=None):
        """Request i becomes a copy of request source[i] (int32 [batch] on the device; itself: it goes on; negative: it
        ends): cache, text and controls. Of those that continue one request the first goes on in its blocks, the others
        get copies; one whose copy the pool does not hold keeps the text and has to run it again (its lens is 0)."""
        torch = self.torch
        if stream is not None:
            with torch.cuda.stream(stream):
                return self.fork(source)
        Y.batch_edit(self.lens, self.whole, self.tables, self.pool, self.free, self.block_size, self.lens_out,
                     self.free_out, source=source, tables_out=self.tables_out, copies=self.copies,
                     n_copies=self.n_copies, prefix_len=self.prefix_len)
        Y.cache_copy(self.caches, self.copies, self.n_copies)
        self.tables.copy_(self.tables_out)
        self.lens.copy_(self.lens_out)
        self.free.copy_(self.free_out)
        # (a source outside the batch ends the request too, and is an error that the status tells)
        of, live = source.clamp(0, self.batch - 1).long(), (source >= 0) & (source < self.batch)
        for t in (self.text, self.prompt, self.repetition, self.presence, self.frequency, self.mask):
            t.copy_(t[of])
        self.said.copy_(self.said[of] * live)

    def _layers(self, T, max_new, tables, lens, starts, prefix_blocks, prefix_len, positions=None, tree=None):
        """The first T of self.tokens through every layer, into self.bx and self.binv; where they are trees' nodes,
        with their positions and masks."""
        h, x, inv, proj = self.bh[:T], self.bx[:T], self.binv[:T], self.bproj[:T]
        q, k, v, query, out = self.bq[:T], self.bk[:T], self.bv[:T], self.bquery[:T], self.bout[:T]
        gate, up, m, a_in = self.bg[:T], self.bu[:T], self.bm[:T], self.ba_in[:T]
        self.embedding.lookup(self.tokens[:T], h)
        before = None
        for L in self.L:
            Y.residual_prepare(h, before, L["in_norm"], S.EPS, x, inv)
            Y.linear([L["q"], L["k"], L["v"]], x, self.bwork, [q, k, v], inv_rms=inv)
            Y.paged_prep(q[:, :, :S.HEAD], k, v, self.slots[:T], self.pos[:T] if positions is None else positions,
                         query, *L["pages"], inv_freq=self.inv_freq, q_norm=L["q_norm"], k_norm=L["k_norm"], eps=S.EPS)
            rest = dict(prefix_blocks=prefix_blocks, prefix_len=prefix_len, gate=q[:, :, S.HEAD:])
            if tree is None:
                Y.prefix_attention(query, *L["pages"], tables, lens, starts, max_new, self.attn_work, out, **rest)
            else:
                Y.tree_attention(query, *L["pages"], tables, lens, starts, max_new, tree, self.attn_work, out, **rest)
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
    st = BatchStack(dev, batch=batch, nodes=8)
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
    # random drafts: what a step that verifies them takes, not what it saves
    for i in range(batch):
        st.draft(i, [(53 * i + 7 * j) % st.vocab for j in range(7)], [0, 0, 1, 1, 2, 3, 4])
    st.new.fill_(8)
    with torch.cuda.stream(stream):
        st.verify(8 * batch, stream)
        t0.record()
        st.verify(8 * batch, stream)
        t1.record()
        torch.cuda.synchronize()
    Y.check(Y.status(stream), "verify")
    print("trees of 8 nodes: %.3f ms a step" % t0.elapsed_time(t1))
    print("request 0:", st.text[0, :int(st.said[0])].tolist()[:16], "...")


if __name__ == "__main__":
    main()
