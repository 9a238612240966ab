"""Operators of a batch that verifies drafted trees and forks its requests, as measured cases.

A draft (a small model, n-grams, extra heads) proposes a tree of tokens for each request; one pass
of the model over all nodes tells which path the model itself would have taken. Answers that share
a beginning (beams, several samples) fork one request into many. Five operators of that loop, over
the paged 16-bit K/V cache whose blocks the batch's plan hands out:

  attn      attention of the nodes over the shared prefix, the request's cached rows and, of the
            new rows, the node's ancestors
  draft     the nodes' ancestor bits and positions from their parents; after the pass, the path
            whose tokens are the model's own choices
  logprobs  log probabilities of given tokens, the entropy and the most likely tokens
  edit      which rows each request keeps, and whose it continues: block tables, the pool, and the
            list of blocks that have to be copied
  move      those copies, and the accepted nodes' rows made adjacent, in every layer's cache

`own` False computes them in plain torch operations, True by the library's calls. Heads of 256
channels, 24 query and 4 key/value heads and 151936 tokens are the decode stack's shapes; the others
are generic.
"""
import itertools
import math
import random
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def _lib():
    if "yasakani-for-mac_b200" not in sys.path:
        sys.path.append("yasakani-for-mac_b200")
    import yskn_b200
    return yskn_b200


# ---------------------------------------------------------------------------- the cases

def listed():
    return [
        # One user's step: a tree of 60 nodes behind a short chat; latency.
        dict(name="attn_one_tree", op="attn", batch=1, nodes=60, prefix=0, rows=2000, q_heads=24, kv_heads=4, head=256,
             dtype="bf16", gate=True, block=64),
        # Odd everything: ragged trees, an odd prefix, small heads, short blocks.
        dict(name="attn_odd_19", op="attn", batch=19, nodes=27, prefix=517, rows=3001, q_heads=16, kv_heads=2, head=128,
             dtype="f16", gate=False, block=16),
        # A serving batch with trees behind a shared document and long texts of their own.
        dict(name="attn_batch_32", op="attn", batch=32, nodes=32, prefix=4096, rows=4096, q_heads=24, kv_heads=4,
             head=256, dtype="bf16", gate=True, block=64),
        # One user's tree.
        dict(name="draft_one_tree", op="draft", batch=1, nodes=60, depth=8, length=2000),
        # The trees of a large batch.
        dict(name="draft_batch_256", op="draft", batch=256, nodes=64, depth=12, length=8000),
        # One answer's next token with twenty alternatives.
        dict(name="logprobs_one_row", op="logprobs", rows=1, vocab=151936, tokens=1, top=20, masked=0.0),
        # An odd vocabulary, whose rows start at any 4-byte boundary, with a grammar; candidates scored.
        dict(name="logprobs_odd_33", op="logprobs", rows=33, vocab=50257, tokens=7, top=5, masked=0.4),
        # All nodes of a batch's trees, or the tokens of a prompt.
        dict(name="logprobs_rows_512", op="logprobs", rows=512, vocab=151936, tokens=1, top=8, masked=0.0),
        # After a verification: every request keeps its accepted rows and gives blocks back.
        dict(name="edit_keep_64", op="edit", batch=64, length=4000, block=64, prefix=1000, fork=0.0, room=1.0),
        # Beam search at a full machine: a third of the requests continue others, not all copies fit.
        dict(name="edit_beams_1024", op="edit", batch=1024, length=1500, block=16, prefix=500, fork=0.35, room=0.9),
        # Accepted paths made adjacent in sixteen layers' caches.
        dict(name="move_paths_64", op="move", kind="paths", batch=64, nodes=16, depth=6, rows=250, caches=32,
             kv_heads=4, head=256, block=64),
        # Forked requests' blocks copied in eight layers' caches.
        dict(name="move_copies_256", op="move", kind="copies", copies=256, caches=16, kv_heads=4, head=256, block=64),
    ]


def _size(rng, lo, hi):
    """A whole number from lo..hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attn", "draft", "logprobs", "edit", "move"])
    if op == "attn":
        head, group, kv_heads = rng.choice([64, 128, 256, 256]), rng.randint(1, 8), rng.randint(1, 4)
        nodes = _size(rng, 1, 128)
        batch = _size(rng, 1, max(1, min(64, 1024 // nodes)))
        keys = int(2e8 / (batch * nodes * group * kv_heads))  # scores as in the largest listed case at most
        prefix = rng.choice([0, _size(rng, 1, max(1, min(8192, keys // 2)))])
        return dict(op=op, batch=batch, nodes=nodes, prefix=prefix,
                    rows=nodes + _size(rng, 1, max(1, min(16384, keys - prefix, 131000 // batch))),
                    q_heads=group * kv_heads, kv_heads=kv_heads, head=head, dtype=rng.choice(["bf16", "f16"]),
                    gate=rng.random() < 0.5, block=rng.choice([16, 32, 64, 128]))
    if op == "draft":
        return dict(op=op, batch=_size(rng, 1, 256), nodes=_size(rng, 1, 64), depth=rng.randint(1, 12),
                    length=_size(rng, 1, 20000))
    if op == "logprobs":
        vocab = _size(rng, 500, 151936)
        return dict(op=op, rows=_size(rng, 1, 512), vocab=vocab, tokens=_size(rng, 1, 16), top=rng.randint(1, 32),
                    masked=rng.choice([0.0, 0.5]))
    if op == "edit":
        block = rng.choice([16, 32, 64, 128])
        return dict(op=op, batch=_size(rng, 1, 1024), length=_size(rng, 1, 90 * block), block=block,
                    prefix=_size(rng, 1, 5000) - 1, fork=rng.choice([0.0, round(rng.uniform(0.1, 0.6), 3)]),
                    room=round(rng.uniform(0.5, 1.0), 3))
    head, kv_heads, block = rng.choice([64, 128, 256]), rng.randint(1, 4), rng.choice([16, 32, 64, 128])
    if rng.random() < 0.5:
        nodes = _size(rng, 2, 64)
        return dict(op=op, kind="paths", batch=_size(rng, 1, 64), nodes=nodes, depth=rng.randint(1, 8),
                    rows=_size(rng, nodes, nodes + 200), caches=2 * rng.randint(1, 8), kv_heads=kv_heads, head=head,
                    block=block)
    return dict(op=op, kind="copies", copies=_size(rng, 1, 256 * 64 // block), caches=2 * rng.randint(1, 8),
                kv_heads=kv_heads, head=head, block=block)


def _rng(case, tag):
    """Random numbers that the case alone fixes (sizes, trees: not the values of tensors)."""
    return random.Random("%s %s" % (tag, sorted((k, v) for k, v in case.items() if k != "name")))


def _lengths(case, tag, n, lo, hi):
    """n whole numbers of lo..hi (ragged, both ends among them)."""
    r = _rng(case, tag)
    got = [r.randint(lo, hi) for _ in range(n)]
    got[0] = hi
    if n > 2:
        got[n // 2] = lo
    return got


def _blocks(n, block):
    return -(-n // block)


def _trees(case):
    """The parents of each request's nodes: node 0 is the request's next token, a later node follows
    one of those before it, as a draft's best paths do (breadth first, 2 to 4 children a node)."""
    r = _rng(case, "trees")
    n = case["nodes"]
    return [[-1] + [r.randint((j - 1) // 4, (j - 1) // 2) for j in range(1, k)]
            for k in _lengths(case, "nodes", case["batch"], max(1, n // 2), n)]


def _ancestors(parents):
    """For each node how many it sees of its tree: its depth and itself."""
    seen = []
    for p in parents:
        seen.append(1 + (seen[p] if p >= 0 else 0))
    return seen


def _attn_rows(case, trees):
    """Own rows of each request, its nodes' among them."""
    extra = _lengths(case, "rows", case["batch"], 0, max(0, case["rows"] - case["nodes"]))
    return [len(t) + e for t, e in zip(trees, extra)]


def _edit_plan(case):
    """(own rows, rows kept, source or None) of each request, before the seed's order."""
    r, B = _rng(case, "edit"), case["batch"]
    rows = _lengths(case, "rows", B, 0, case["length"])
    if case["fork"] == 0.0:
        return rows, [max(0, n - r.randint(0, min(64, n))) for n in rows], None
    source = [r.randrange(B) if r.random() < case["fork"] else i for i in range(B)]
    source = [-1 if r.random() < 0.05 else j for j in source]
    keep = [max(0, rows[j] - (r.randint(0, 3) if r.random() < 0.3 else 0)) if j >= 0 else 0 for j in source]
    return rows, keep, source


def _edit_counts(case):
    """(held, kept blocks, blocks copied, table width) of a batch."""
    rows, keep, source = _edit_plan(case)
    bs = case["block"]
    held, kept = [_blocks(n, bs) for n in rows], [_blocks(n, bs) for n in keep]
    copied = 0
    if source is not None:
        best = {}
        for i, j in enumerate(source):
            if j >= 0 and (j not in best or keep[i] > keep[best[j]]):
                best[j] = i
        copied = sum(kept[i] for i, j in enumerate(source) if j >= 0 and best[j] != i)
    return held, kept, copied, max(1, max(held))


def work(case):
    op = case["op"]
    if op == "attn":
        trees = _trees(case)
        rows = _attn_rows(case, trees)
        P, D, hq, hk = case["prefix"], case["head"], case["q_heads"], case["kv_heads"]
        tokens = sum(len(t) for t in trees)
        kv = (P + sum(rows)) * hk * D * 2 * 2
        seen = sum(len(t) * (P + n - len(t)) + sum(_ancestors(t)) for t, n in zip(trees, rows))
        heads = tokens * hq * D * 2 * (3 if case["gate"] else 2)
        return {"bytes": float(kv + heads + tokens * _blocks(case["nodes"], 8)),
                "flops": float(4 * seen * hq * D)}
    if op == "draft":
        tokens = sum(len(t) for t in _trees(case))
        # parents, drafted tokens and choices in; bits and positions out; per request its path
        return {"bytes": float(tokens * (4 * 3 + 4 + 4 * _blocks(case["nodes"], 32)) +
                               case["batch"] * (4 * 6 + 4 * case["depth"])), "flops": 0.0}
    if op == "logprobs":
        M, V = case["rows"], case["vocab"]
        return {"bytes": float(4 * M * V + M * (8 * case["tokens"] + 4 + 8 * case["top"])), "flops": float(4 * M * V)}
    if op == "edit":
        held, kept, copied, _ = _edit_counts(case)
        B = case["batch"]
        back = max(0, sum(held) - sum(kept) + copied)
        moved = 8 * sum(kept) + 20 * copied if case["fork"] else 0
        return {"bytes": float(B * 16 + moved + 8 * back), "flops": 0.0}
    row = case["kv_heads"] * case["head"] * 2 * case["caches"]
    if case["kind"] == "copies":
        rows = sum(_lengths(case, "copy", case["copies"], 1, case["block"]))
    else:
        rows = sum(max(0, len(p) - 1) for p in _paths(case, _trees(case)))
    return {"bytes": float(2 * rows * row), "flops": 0.0}


# ---------------------------------------------------------------------------- the inputs

def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEV)


def _i32(*shape):
    return torch.empty(shape, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    order = list(range(case.get("batch", 1)))
    random.Random(seed).shuffle(order)
    s = {"case": case}
    {"attn": _prepare_attn, "draft": _prepare_draft, "logprobs": _prepare_logprobs, "edit": _prepare_edit,
     "move": _prepare_move}[case["op"]](case, g, order, s)
    return s


def _randn(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def _tree_bits(trees, words):
    """Ancestor bits [nodes of all trees][words], as the draft operator writes them."""
    rows = []
    for parents in trees:
        bits = []
        for j, p in enumerate(parents):
            bits.append((bits[p] if p >= 0 else 0) | 1 << j)
        rows += bits
    signed = lambda w: w - 2 ** 32 if w >= 2 ** 31 else w  # noqa: E731
    return _ints([[signed(b >> 32 * w & 0xffffffff) for w in range(words)] for b in rows])


def _tables(g, held, spare=1):
    """Block tables of the batch (numbers in any order), the numbers that are left, and how many blocks."""
    B, width, n = len(held), max(1, max(held)), sum(held) + spare
    numbers = torch.randperm(n, generator=g, device=DEV).to(torch.int32)
    tables = torch.full((B, width), -1, dtype=torch.int32, device=DEV)
    at = torch.arange(width, device=DEV)[None, :] < _ints(held, torch.int64)[:, None]
    tables[at] = numbers[:sum(held)]
    return tables, numbers[sum(held):], n


def _prepare_attn(case, g, order, s):
    trees = _trees(case)
    rows = _attn_rows(case, trees)
    trees, rows = [trees[i] for i in order], [rows[i] for i in order]
    P, D, bs, hq, hk = case["prefix"], case["head"], case["block"], case["q_heads"], case["kv_heads"]
    dt, T, pre = DTYPES[case["dtype"]], sum(len(t) for t in trees), _blocks(P, bs)
    tables, rest, n_blocks = _tables(g, [_blocks(n, bs) for n in rows], pre + 1)
    s.update(q=_randn(g, (T, hq, D), dt, 1.5), gate=_randn(g, (T, hq, D), dt, 2.0) if case["gate"] else None,
             k_cache=_randn(g, (n_blocks, hk, bs, D), dt).transpose(1, 2),
             v_cache=_randn(g, (n_blocks, hk, bs, D), dt).transpose(1, 2), tables=tables,
             lens=_ints([P + n for n in rows]),
             starts=_ints(list(itertools.accumulate((len(t) for t in trees), initial=0))),
             prefix_blocks=rest[:pre].clone(), prefix=P, max_new=case["nodes"],
             bits=_tree_bits(trees, _blocks(case["nodes"], 32)), out=torch.empty((T, hq, D), dtype=dt, device=DEV),
             work=None)


def _prepare_draft(case, g, order, s):
    trees = _trees(case)
    trees = [trees[i] for i in order]
    lens = _lengths(case, "lens", case["batch"], 0, case["length"])
    counts, T, words, vocab = [len(t) for t in trees], sum(len(t) for t in trees), _blocks(case["nodes"], 32), 1000
    tokens = torch.randint(0, vocab, (T,), generator=g, device=DEV, dtype=torch.int32)
    choice = torch.randint(0, vocab, (T,), generator=g, device=DEV, dtype=torch.int32)
    # the model agrees with the draft at most nodes: its choice there is one of the node's children
    starts = list(itertools.accumulate(counts, initial=0))
    child = list(range(T))
    for s0, parents in zip(starts, trees):
        for j, p in enumerate(parents):
            if p >= 0:
                child[s0 + p] = s0 + j  # its last one
    child = _ints(child, torch.int64)
    agrees = torch.rand(T, generator=g, device=DEV) < 0.85
    choice = torch.where(agrees, tokens[child], choice)
    B = case["batch"]
    s.update(parents=_ints([p for t in trees for p in t]), tokens=tokens, choice=choice, starts=_ints(starts),
             requests=_ints([i for i, n in enumerate(counts) for _ in range(n)]),
             lens=_ints([lens[i] + n for i, n in zip(order, counts)]), mask=_i32(T, words), positions=_i32(T),
             path=_i32(B, case["depth"]), accepted=_i32(B), lens_out=_i32(B), next=_i32(B), max_new=case["nodes"])


def _prepare_logprobs(case, g, order, s):
    M, V, n = case["rows"], case["vocab"], case["tokens"]
    # from sure rows to undecided ones; every other row as a 16-bit head would give it, with ties
    x = torch.randn((M, V), generator=g, device=DEV) * (0.5 + 4 * torch.rand((M, 1), generator=g, device=DEV))
    x[::2] = x[::2].bfloat16().float()
    if case["masked"]:
        x[torch.rand((M, V), generator=g, device=DEV) < case["masked"]] = -math.inf
    tokens = torch.randint(0, V, (M, n), generator=g, device=DEV)
    tokens[:, 0] = x.argmax(1)  # the answer's own token, then others that are allowed
    tokens = torch.where(x.gather(1, tokens) == -math.inf, tokens[:, :1], tokens).to(torch.int32)
    f32 = lambda *shape: torch.empty(shape, device=DEV)  # noqa: E731
    s.update(logits=x, tokens=tokens, logprobs=f32(M, n), entropy=f32(M), top_logprobs=f32(M, min(case["top"], V)),
             top_ids=_i32(M, min(case["top"], V)))


def _prepare_edit(case, g, order, s):
    rows, keep, source = _edit_plan(case)
    held, _, copied, _ = _edit_counts(case)
    B, P, bs = case["batch"], case["prefix"], case["block"]
    place = {i: k for k, i in enumerate(order)}  # the seed's order of the requests
    rows, keep, held = ([x[i] for i in order] for x in (rows, keep, held))
    if source is not None:
        source = [place[source[i]] if source[i] >= 0 else -1 for i in order]
    free = max(1, int(copied * case["room"]))
    tables, rest, n_blocks = _tables(g, held, free)
    pool = torch.full((n_blocks,), -1, dtype=torch.int32, device=DEV)
    pool[:free] = rest
    s.update(lens=_ints([P + n if n else 0 for n in rows]), keep=_ints([P + n if n else 0 for n in keep]),
             source=None if source is None else _ints(source), tables=tables, pool=pool, free=_ints([free]), block=bs,
             prefix=P, lens_out=_i32(B), free_out=_i32(1), tables_out=tables.clone(),
             copies=_i32(3, max(1, copied + 3)), n_copies=_i32(1))


def _paths(case, trees):
    """An accepted path of each tree: up to `depth` nodes, those after node 0 behind the places that the
    path's rows go to (so that a pass can be repeated)."""
    r, paths = _rng(case, "paths"), []
    for parents in trees:
        want, path = min(case["depth"], len(parents)), [0]
        for j in range(1, len(parents)):
            if len(path) < want and j >= want and r.random() < 0.5:
                path.append(j)
        paths.append(path)
    return paths


def _prepare_move(case, g, order, s):
    hk, D, bs = case["kv_heads"], case["head"], case["block"]
    if case["kind"] == "copies":
        n = case["copies"]
        n_blocks = 2 * n + 1
        numbers = torch.randperm(n_blocks, generator=g, device=DEV).to(torch.int32)
        source = numbers[torch.randint(0, n, (n,), generator=g, device=DEV)]  # several copies of one block
        rows = _ints(_lengths(case, "copy", n, 1, bs))
        s.update(copies=torch.stack([source, numbers[n:2 * n], rows]).contiguous(), n_copies=_ints([n]))
    else:
        trees = _trees(case)
        paths, rows = _paths(case, trees), _lengths(case, "rows", case["batch"], 0, case["rows"])
        trees, paths, rows = ([x[i] for i in order] for x in (trees, paths, rows))
        ends = [n + len(t) for n, t in zip(rows, trees)]
        tables, _, n_blocks = _tables(g, [_blocks(n, bs) for n in ends])
        width = case["depth"]
        s.update(tables=tables, lens=_ints(ends), path=_ints([p + [-1] * (width - len(p)) for p in paths]),
                 starts=_ints(list(itertools.accumulate((len(t) for t in trees), initial=0))))
    # 16-bit patterns that are numbers of either type
    s["pools"] = [torch.randint(0, 0x3c00, (n_blocks, hk, bs, D), generator=g, device=DEV, dtype=torch.int16)
                  for _ in range(case["caches"])]
    s["caches"], s["set"] = [c.view(torch.bfloat16).transpose(1, 2) for c in s["pools"]], None


# ------------------------------------------------------------------------------ the pass

def run(s):
    form = _OWN if own else _PLAIN
    return form[s["case"]["op"]](s)


def _own_attn(s):
    Y = _lib()
    if s["work"] is None:
        n = Y.prefix_attention_work_bytes(s["q"].shape[0], s["tables"].shape[0], s["max_new"], s["q"].shape[1],
                                          s["k_cache"].shape[2], s["q"].shape[2])
        s["work"] = torch.empty(n, dtype=torch.uint8, device=DEV)
    Y.tree_attention(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["lens"], s["starts"], s["max_new"], s["bits"],
                     s["work"], s["out"], prefix_blocks=s["prefix_blocks"], prefix_len=s["prefix"], gate=s["gate"])
    return s["out"]


def _plain_attn(s):
    q, kc, vc, P, n_max = s["q"].float(), s["k_cache"], s["v_cache"], s["prefix"], s["max_new"]
    (T, hq, D), hk, B = q.shape, kc.shape[2], s["tables"].shape[0]
    G = hq // hk
    starts, lens = s["starts"].long(), s["lens"].long()
    n = starts[1:] - starts[:-1]
    # nodes padded to n_max a request: [B][hk][n_max * G][D]
    j = torch.arange(n_max, device=q.device)
    token = (starts[:-1, None] + j[None, :]).clamp(max=T - 1)
    qp = q[token].view(B, n_max, hk, G, D).permute(0, 2, 1, 3, 4).reshape(B, hk, n_max * G, D)
    flat = lambda c, t: c[t.clamp(min=0).long()].flatten(-4, -3).float()  # noqa: E731  blocks -> rows [..][hk][D]
    kp, vp = (flat(c, s["prefix_blocks"])[:P].transpose(0, 1) for c in (kc, vc))  # [hk][P][D]
    ko, vo = (flat(c, s["tables"]).transpose(1, 2) for c in (kc, vc))  # [B][hk][width * block][D]
    row = torch.arange(ko.shape[2], device=q.device)
    vo = torch.where((P + row < lens[:, None])[:, None, :, None], vo, 0.0)
    # a node sees every row before the request's new ones, and of those its ancestors and itself
    new = P + row - (lens - n)[:, None]  # [B][rows]: which new row, negative before them
    at = new.clamp(0, 32 * s["bits"].shape[1] - 1)
    words = s["bits"][token].gather(2, (at >> 5)[:, None, :].expand(B, n_max, -1))  # [B][n_max][rows]
    sees = ((words >> (at & 31)[:, None, :]) & 1 == 1) & (new < n[:, None])[:, None, :] | (new < 0)[:, None, :]
    scale = 1.0 / math.sqrt(D)
    sp = torch.matmul(qp, kp.transpose(-1, -2)[None]).mul_(scale).view(B, hk, n_max, G, P)
    so = torch.matmul(qp, ko.transpose(-1, -2)).mul_(scale).view(B, hk, n_max, G, -1)
    so.masked_fill_(~sees[:, None, :, None, :], -math.inf)
    top = so.amax(-1, keepdim=True)
    if P:
        top = torch.maximum(top, sp.amax(-1, keepdim=True))
    top = torch.where(top == -math.inf, 0.0, top)
    sp.sub_(top).exp_()
    so.sub_(top).exp_()
    den = sp.sum(-1) + so.sum(-1)
    num = torch.matmul(sp.view(B, hk, n_max * G, P), vp[None]) + torch.matmul(so.view(B, hk, n_max * G, -1), vo)
    out = num.view(B, hk, n_max, G, D) / torch.where(den > 0, den, 1.0)[..., None]
    out = out.permute(0, 2, 1, 3, 4).reshape(B, n_max, hq, D)
    t = torch.arange(T, device=q.device)
    r = torch.searchsorted(starts[1:], t, right=True)
    out = out[r, t - starts[r]]
    if s["gate"] is not None:
        out = out * torch.sigmoid(s["gate"].float())
    return out.to(s["q"].dtype)


def _own_draft(s):
    Y = _lib()
    Y.tree_plan(s["parents"], s["requests"], s["starts"], s["lens"], s["mask"], s["positions"])
    Y.tree_accept(s["tokens"], s["parents"], s["choice"], s["starts"], s["lens"], s["path"], s["accepted"],
                  s["lens_out"], s["next"])
    return s["mask"], s["positions"], s["path"], s["accepted"], s["lens_out"], s["next"]


def _plain_draft(s):
    parents, starts, lens = s["parents"].long(), s["starts"].long(), s["lens"].long()
    T, words = s["mask"].shape
    B, width = s["path"].shape
    r = s["requests"].long()
    local = torch.arange(T, device=DEV) - starts[r]
    bit = torch.arange(32 * words, device=DEV)
    seen = bit[None, :] == local[:, None]
    up, depth = torch.where(parents >= 0, parents, -1), torch.zeros_like(parents)
    for _ in range(s["max_new"] - 1):  # one more ancestor a round
        seen |= bit[None, :] == up[:, None]
        depth += up >= 0
        up = torch.where(up >= 0, parents[(starts[r] + up).clamp(min=0)], -1)
    mask = (seen.view(T, words, 32).long() << torch.arange(32, device=DEV)).sum(-1)
    mask = torch.where(mask >= 2 ** 31, mask - 2 ** 32, mask).to(torch.int32)
    n = starts[1:] - starts[:-1]
    positions = (lens - n)[r] + depth
    # the path: node 0, then in order every node that follows the last one and is its choice
    path = torch.full((B, width), -1, dtype=torch.int64, device=DEV)
    last, count = torch.zeros_like(n), (n > 0).long()
    path[:, 0] = torch.where(n > 0, 0, -1)
    for j in range(1, s["max_new"]):
        at = (starts[:-1] + j).clamp(max=T - 1)
        choice = s["choice"].long()[(starts[:-1] + last).clamp(max=T - 1)]
        takes = (j < n) & (parents[at] == last) & (s["tokens"].long()[at] == choice) & (choice >= 0) & (count < width)
        put = torch.where(takes, count, width - 1)[:, None]
        path.scatter_(1, put, torch.where(takes[:, None], j, path.gather(1, put)))
        last, count = torch.where(takes, j, last), count + takes
    nxt = torch.where(n > 0, s["choice"].long()[(starts[:-1] + last).clamp(max=T - 1)], -1)
    i32 = lambda x: x.to(torch.int32)  # noqa: E731
    return mask, i32(positions), i32(path), i32(count), i32(lens - n + count), i32(nxt)


def _own_logprobs(s):
    _lib().token_logprobs(s["logits"], s["tokens"], s["logprobs"], entropy=s["entropy"],
                          top_logprobs=s["top_logprobs"], top_ids=s["top_ids"])
    return s["logprobs"], s["entropy"], s["top_logprobs"], s["top_ids"]


def _plain_logprobs(s):
    x, k = s["logits"], s["top_ids"].shape[1]
    # equal logits: the lowest token first; -0 and 0 are equal
    bits = (x + 0.0).view(torch.int32).long()
    key = torch.where(bits >= 0, bits, -(bits & 0x7fffffff)) * 2 ** 32 - torch.arange(x.shape[1], device=x.device)
    ids = key.topk(k, dim=1).indices
    top = x.gather(1, ids[:, :1])
    d = x - top
    p = d.exp().scatter_(1, ids[:, :1], 0.0)  # all but the most likely one, whose weight is 1
    rest = p.sum(1, keepdim=True)
    log_sum = torch.log1p(rest)
    entropy = log_sum - torch.where(p > 0, p * d, 0.0).sum(1, keepdim=True) / (1.0 + rest)
    logprobs = d.gather(1, s["tokens"].long()) - log_sum
    return logprobs, entropy[:, 0], d.gather(1, ids) - log_sum, ids.to(torch.int32)


def _own_edit(s):
    fork = {} if s["source"] is None else dict(source=s["source"], tables_out=s["tables_out"], copies=s["copies"],
                                               n_copies=s["n_copies"])
    _lib().batch_edit(s["lens"], s["keep"], s["tables"], s["pool"], s["free"], s["block"], s["lens_out"], s["free_out"],
                      prefix_len=s["prefix"], **fork)
    if s["source"] is None:
        return s["lens_out"], s["free_out"], s["pool"]
    return s["lens_out"], s["free_out"], s["pool"], s["tables_out"], s["copies"], s["n_copies"]


def _plain_edit(s):
    bs, P, pool, tables = s["block"], s["prefix"], s["pool"], s["tables"]
    lens, keep, free = s["lens"].long(), s["keep"].long(), s["free"].long()
    B, width = tables.shape
    i = torch.arange(B, device=DEV)
    source = i if s["source"] is None else s["source"].long()
    real = source >= 0
    source = source.clamp(min=0)
    length = torch.where(real, torch.minimum(keep.clamp(min=0), lens[source]), 0)
    own_rows = (length - P).clamp(min=0)
    kept, held = (own_rows + bs - 1) // bs, ((lens - P).clamp(min=0) + bs - 1) // bs
    # of the requests that continue j, the one that keeps most rows (the lowest number) has j's blocks
    rank = torch.where(real, length * B + (B - 1 - i), -1)
    best = torch.full((B,), -1, dtype=torch.int64, device=DEV).scatter_reduce(0, source, rank, "amax")
    heir = real & (best[source] == rank)
    stays = torch.zeros_like(held).scatter_add(0, source, torch.where(heir, kept, 0))
    back = held - stays
    back_end = back.cumsum(0)
    need = torch.where(real & ~heir, kept, 0)
    have = free + back_end[-1]
    room = have if s["source"] is None else have.clamp(max=s["copies"].shape[1])
    served = need.cumsum(0) <= room
    need = torch.where(served, need, 0)
    length = torch.where(served | (kept == 0) | heir, length, 0)
    left = have - need.sum()
    at = torch.arange(pool.numel(), device=DEV)
    giver = torch.searchsorted(back_end, at - free, right=True).clamp(max=B - 1)
    place = (stays[giver] + at - free - (back_end - back)[giver]).clamp(0, width - 1)
    stack = torch.where((at >= free) & (at < have), tables[giver, place], pool)
    i32 = lambda x: x.to(torch.int32)  # noqa: E731
    pool_out = torch.where((at >= free) & (at < left), stack, pool)
    if s["source"] is None:
        return i32(length), i32(left), pool_out
    first = need.cumsum(0) - need  # copies before the request's
    col = torch.arange(width, device=DEV)[None, :]
    taken = stack[(have - 1 - first[:, None] - col).clamp(0, pool.numel() - 1)]
    fresh = col < need[:, None]
    tables_out = torch.where(heir[:, None] & (col < kept[:, None]), tables[source],
                             torch.where(fresh, taken, s["tables_out"]))
    # entry by entry into the list; what is no copy goes to a place behind its end
    room = s["copies"].shape[1]
    at = torch.where(fresh, first[:, None] + col, room).flatten()
    copies = torch.full((3, room + 1), -1, dtype=torch.int32, device=DEV)
    copies[2] = 0
    for row, value in enumerate((tables[source], taken, (own_rows[:, None] - col * bs).clamp(max=bs))):
        copies[row].scatter_(0, at, i32(value).flatten())
    copies = copies[:, :room]
    return i32(length), i32(left), pool_out, tables_out, copies, i32(need.sum()[None])


def _own_move(s):
    Y = _lib()
    if s["set"] is None:
        s["set"] = Y.CacheSet(s["caches"])
    if s["case"]["kind"] == "copies":
        Y.cache_copy(s["set"], s["copies"], s["n_copies"])
    else:
        Y.cache_compact(s["set"], s["tables"], s["lens"], s["starts"], s["path"])
    return s["pools"]


def _plain_move(s):
    bs = s["pools"][0].shape[2]
    if s["case"]["kind"] == "copies":
        source, target, rows = (x.long() for x in s["copies"])
        moved = (torch.arange(bs, device=DEV)[None, :] < rows[:, None])[:, None, :, None]
        for c in s["pools"]:
            c[target] = torch.where(moved, c[source], c[target])
        return s["pools"]
    n = (s["starts"][1:] - s["starts"][:-1]).long()
    base, path = s["lens"].long() - n, s["path"].long()
    k = torch.arange(path.shape[1], device=DEV)[None, :]
    i = torch.arange(path.shape[0], device=DEV)[:, None]
    source, target = base[:, None] + path.clamp(min=0), base[:, None] + torch.where(path >= 0, k, 0)  # none: itself
    for c in s["pools"]:
        c[s["tables"][i, target // bs].long(), :, target % bs] = c[s["tables"][i, source // bs].long(), :, source % bs]
    return s["pools"]


_OWN = {"attn": _own_attn, "draft": _own_draft, "logprobs": _own_logprobs, "edit": _own_edit, "move": _own_move}
_PLAIN = {"attn": _plain_attn, "draft": _plain_draft, "logprobs": _plain_logprobs, "edit": _plain_edit,
          "move": _plain_move}


# ------------------------------------------------------------- the definitions in 64 bits

def exact(case, seed):
    f64 = torch.float64
    if case["op"] == "attn":
        s = prepare(case, seed)
        P, (T, hq, D), hk = s["prefix"], s["q"].shape, s["k_cache"].shape[2]
        G, bs = hq // hk, case["block"]
        lens, starts = s["lens"].tolist(), s["starts"].tolist()
        out = torch.zeros((T, hq, D), dtype=f64, device=DEV)
        for b, length in enumerate(lens):
            t0, t1 = starts[b], starts[b + 1]
            ids = s["tables"][b, :_blocks(length - P, bs)].long()
            k, v = (torch.cat([c[s["prefix_blocks"].long()].reshape(-1, hk, D)[:P],
                               c[ids].reshape(-1, hk, D)[:length - P]]).to(f64) for c in (s["k_cache"], s["v_cache"]))
            hidden = torch.zeros((t1 - t0, length), dtype=torch.bool, device=DEV)
            for j in range(t1 - t0):
                hidden[:, length - (t1 - t0) + j] = (s["bits"][t0:t1, j // 32] >> (j % 32)) % 2 == 0
            for h in range(hk):
                q = s["q"][t0:t1, h * G:(h + 1) * G].to(f64)  # [n][G][D]
                w = torch.einsum("ngd,ld->gnl", q, k[:, h]) / math.sqrt(D)
                w = torch.softmax(w.masked_fill(hidden[None], -math.inf), -1)
                out[t0:t1, h * G:(h + 1) * G] = torch.einsum("gnl,ld->ngd", w, v[:, h])
        if s["gate"] is not None:
            out = out / (1 + torch.exp(-s["gate"].to(f64)))
        return out
    if case["op"] == "logprobs":
        s = prepare(case, seed)
        M, k = s["top_ids"].shape
        logprobs, entropy = torch.zeros_like(s["logprobs"], dtype=f64), torch.zeros(M, dtype=f64, device=DEV)
        tops, ids = torch.zeros((M, k), dtype=f64, device=DEV), torch.zeros((M, k), dtype=torch.int32, device=DEV)
        for m in range(M):
            x = s["logits"][m].to(f64)
            order = torch.sort(x, descending=True, stable=True)
            # the others' sum beside the first one's 1, so that a sure row keeps its small numbers
            log_z = torch.log1p(torch.exp(order.values[1:] - order.values[0]).sum())
            logp = (x - order.values[0]) - log_z
            p = logp.exp()
            logprobs[m] = logp[s["tokens"][m].long()]
            entropy[m] = -(p * logp.clamp(min=-1e300)).sum()
            tops[m], ids[m] = logp[order.indices[:k]], order.indices[:k].to(torch.int32)
        return logprobs, entropy, tops, ids
    return None  # whole numbers and copies: held equal
