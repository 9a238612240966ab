"""The operators of a batch that shares a prompt prefix, as measured cases.

Four operators make one decode, verification or prompt step of a batch whose requests begin
with the same rows (a system prompt, a document, examples), over a paged 16-bit K/V cache:

  plan    blocks, slots and positions of the step's new tokens from the request lengths
  prep    query and key heads normalised and rotated by one or three position axes, new key
          and value rows into the cache
  attn    attention of all rows over the shared prefix, read once for the batch, and each
          request's own rows
  logits  penalties for repeated tokens, biases and a grammar mask on the head's logits

`own` False computes them in plain torch operations, True by the library's calls. Heads of
256 channels, 24 query and 4 key/value heads, 64 rotated channels and 151936 tokens are the
decode stack's shapes; the others are generic.
"""
import itertools
import math
import random
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6


def _lib():
    if "yasakani-for-mac_b200" not in sys.path:
        sys.path.append("yasakani-for-mac_b200")
    import yskn_b200
    return yskn_b200


# ---------------------------------------------------------------------------- the cases

def listed():
    return [
        # One decode step of a serving batch: a token for each of 256 requests.
        dict(name="plan_decode_256", op="plan", batch=256, new=1, length=8192, block=64, prefix=4096, ended=0.02,
             room=1.0),
        # Prompts arriving at a full machine: ragged new tokens, the pool too small for all.
        dict(name="plan_prompts_4096", op="plan", batch=4096, new=300, length=2000, block=16, prefix=1000, ended=0.1,
             room=0.9),
        # The smallest step: one request's token, from the projections' f32 rows with gates.
        dict(name="prep_one_token", op="prep", tokens=1, q_heads=24, kv_heads=4, head=256, rot=64, axes=1,
             source="f32", dtype="bf16", gate=True, norm=True, block=64),
        # A prompt chunk of text and images: three position axes.
        dict(name="prep_prompt_8192", op="prep", tokens=8192, q_heads=24, kv_heads=4, head=256, rot=64, axes=3,
             source="f32", dtype="bf16", gate=True, norm=True, block=64),
        # Odd token count, small heads rotated whole, 16-bit projections.
        dict(name="prep_odd_1037", op="prep", tokens=1037, q_heads=20, kv_heads=5, head=128, rot=128, axes=3,
             source="f16", dtype="f16", gate=False, norm=True, block=16),
        # Two requests behind a short prompt: latency.
        dict(name="attn_two_requests", op="attn", batch=2, new=1, prefix=512, own_rows=60, q_heads=24, kv_heads=4,
             head=256, dtype="bf16", gate=True, block=64),
        # Speculative verification: a few rows for each request, an odd prefix, small heads.
        dict(name="attn_verify_19", op="attn", batch=19, new=8, prefix=8191, own_rows=700, q_heads=16, kv_heads=2,
             head=128, dtype="f16", gate=False, block=16),
        # Decode at the long context: 64 requests behind 32k shared rows.
        dict(name="attn_decode_64", op="attn", batch=64, new=1, prefix=32768, own_rows=1024, q_heads=24, kv_heads=4,
             head=256, dtype="bf16", gate=True, block=64),
        # Prompt chunks of 16 requests behind a shared document.
        dict(name="attn_prompts_16", op="attn", batch=16, new=512, prefix=8192, own_rows=900, q_heads=24, kv_heads=4,
             head=256, dtype="bf16", gate=True, block=64),
        # One request's logits with everything on.
        dict(name="logits_one_row", op="logits", rows=1, vocab=151936, history=512, biases=16, mask=True),
        # An odd vocabulary, whose rows start at any 4-byte boundary; no mask.
        dict(name="logits_odd_33", op="logits", rows=33, vocab=50257, history=4000, biases=300, mask=False),
        # A whole batch with long histories and grammars.
        dict(name="logits_batch_256", op="logits", rows=256, vocab=151936, history=16384, biases=64, mask=True),
    ]


def _size(rng, lo, hi):
    """A whole number from lo..hi, spread over its logarithm."""
    n = min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))
    return n + 1 if n == 3072 else n


def draw(rng):
    op = rng.choice(["plan", "prep", "attn", "logits"])
    if op == "plan":
        batch = _size(rng, 1, 4096)
        return dict(op=op, batch=batch, new=_size(rng, 1, max(1, min(8192, 1000000 // batch))),
                    length=_size(rng, 1, 20000), block=rng.choice([16, 32, 64, 128]), prefix=_size(rng, 1, 9000) - 1,
                    ended=round(rng.uniform(0.0, 0.3), 3), room=round(rng.uniform(0.5, 1.0), 3))
    if op == "prep":
        head = rng.choice([64, 128, 256])
        group, kv_heads = rng.randint(1, 8), rng.randint(1, 6)
        source = rng.choice(["f32", "f32", "bf16", "f16"])
        return dict(op=op, tokens=_size(rng, 1, 8192 * 28 // (kv_heads * (group + 2)) * 256 // head // 3),
                    q_heads=group * kv_heads, kv_heads=kv_heads, head=head,
                    rot=rng.choice([r for r in (32, 64, 96, 128, 256) if r <= head]), axes=rng.choice([1, 3]),
                    source=source, dtype="bf16" if source == "f32" else source, gate=rng.random() < 0.5,
                    norm=rng.random() < 0.8, block=rng.choice([16, 32, 64, 128]))
    if op == "attn":
        head = rng.choice([64, 128, 256, 256])
        group, kv_heads = rng.randint(1, 8), rng.randint(1, 4)
        new = rng.choice([1, 1, _size(rng, 1, 16), _size(rng, 1, 256)])
        batch = _size(rng, 1, max(1, min(128, 4096 // new)))
        keys = int(9e8 / (batch * new * group * kv_heads)) - 900  # scores as in the largest listed case at most
        return dict(op=op, batch=batch, new=new, prefix=_size(rng, 1, max(1, min(32769, keys))) - 1,
                    own_rows=_size(rng, new, max(new, 900)), q_heads=group * kv_heads, kv_heads=kv_heads, head=head,
                    dtype=rng.choice(["bf16", "f16"]), gate=rng.random() < 0.5, block=rng.choice([16, 32, 64, 128]))
    rows = _size(rng, 1, 256)
    return dict(op=op, rows=rows, vocab=_size(rng, 500, 151936), history=_size(rng, 1, 16384),
                biases=_size(rng, 1, 301) - 1, mask=rng.random() < 0.5)


def _lengths(case, tag, n, lo, hi):
    """n whole numbers of lo..hi that the case alone fixes (ragged, both ends among them)."""
    r = random.Random("%s %s" % (tag, sorted((k, v) for k, v in case.items() if k != "name")))
    got = [r.randint(lo, hi) for _ in range(n)]
    got[0] = hi
    if n > 2:
        got[n // 2] = lo
    return got


def _plan_lengths(case):
    """(length, new) of each request: own rows and new tokens; new -1 for an ended one."""
    B, r = case["batch"], random.Random("ended %s" % sorted((k, v) for k, v in case.items() if k != "name"))
    own_rows = _lengths(case, "own", B, 0, case["length"])
    new = _lengths(case, "new", B, 1, case["new"])
    return own_rows, [-1 if r.random() < case["ended"] else 0 if r.random() < 0.02 else n for n in new]


def _blocks(n, block):
    return -(-n // block)


def _plan_sizes(case):
    """(table width, new tokens in all, blocks held, blocks needed) of a plan."""
    own_rows, new = _plan_lengths(case)
    bs = case["block"]
    held = sum(_blocks(o, bs) for o in own_rows)
    need = sum(_blocks(o + n, bs) - _blocks(o, bs) for o, n in zip(own_rows, new) if n > 0)
    width = max(_blocks(o + max(n, 0), bs) for o, n in zip(own_rows, new))
    return width, sum(max(n, 0) for n in new), held, need


def _attn_lengths(case):
    """(new tokens, own rows with them) of each request."""
    B, n = case["batch"], case["new"]
    new = _lengths(case, "new", B, min(n, max(1, n // 8)), n)
    extra = _lengths(case, "own", B, 0, max(0, case["own_rows"] - n))
    return new, [a + b for a, b in zip(new, extra)]


def work(case):
    op = case["op"]
    if op == "plan":
        width, tokens, held, need = _plan_sizes(case)
        # lengths in and out, new lengths, starts; per token slot, position and request; per
        # new block its number from the pool and into the table, per token block its number
        return {"bytes": 16.0 * case["batch"] + 16.0 * tokens + 8.0 * need, "flops": 0.0}
    if op == "prep":
        T, D, src = case["tokens"], case["head"], 4 if case["source"] == "f32" else 2
        heads = case["q_heads"] + 2 * case["kv_heads"]
        return {"bytes": float(T * heads * D * (src + 2) + T * (8 + 4 * case["axes"])),
                "flops": float(T * heads * D * 6)}
    if op == "attn":
        new, rows = _attn_lengths(case)
        P, D, hq, hk = case["prefix"], case["head"], case["q_heads"], case["kv_heads"]
        tokens = sum(new)
        kv = (P + sum(rows)) * hk * D * 2 * 2
        seen = sum(n * (P + o) - n * (n - 1) // 2 for n, o in zip(new, rows))
        return {"bytes": float(kv + tokens * hq * D * 2 * (3 if case["gate"] else 2)),
                "flops": float(4 * seen * hq * D)}
    M, V = case["rows"], case["vocab"]
    hist = sum(_lengths(case, "history", M, 0, case["history"]))
    return {"bytes": float(8 * M * V + (M * V / 8 if case["mask"] else 0) + 4 * hist + 8 * M * case["biases"]),
            "flops": float(4 * M * V)}


# ---------------------------------------------------------------------------- the inputs

def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    order = list(range(case.get("batch", case.get("rows", 1))))
    random.Random(seed).shuffle(order)
    s = {"case": case}
    {"plan": _prepare_plan, "prep": _prepare_prep, "attn": _prepare_attn, "logits": _prepare_logits}[case["op"]](
        case, g, order, s)
    return s


def _prepare_plan(case, g, order, s):
    own_rows, new = _plan_lengths(case)
    own_rows, new = [own_rows[i] for i in order], [new[i] for i in order]
    B, bs, P = case["batch"], case["block"], case["prefix"]
    width, tokens, held, need = _plan_sizes(case)
    free = max(1, int(need * case["room"]))
    numbers = torch.randperm(held + free, generator=g, device=DEV).to(torch.int32)
    counts = _ints([_blocks(o, bs) for o in own_rows], torch.int64)
    tables = torch.full((B, width), -1, dtype=torch.int32, device=DEV)
    at = torch.arange(width, device=DEV)[None, :] < counts[:, None]
    tables[at] = numbers[:held]
    pool = torch.full((held + free,), -1, dtype=torch.int32, device=DEV)
    pool[:free] = numbers[held:]
    i32 = lambda n: torch.empty(n, dtype=torch.int32, device=DEV)  # noqa: E731
    s.update(lens=_ints([P + o if o else 0 for o in own_rows]), new=_ints(new), tables=tables, pool=pool,
             free=_ints([free]), block=bs, prefix=P, tokens=tokens + 5, lens_out=i32(B), free_out=i32(1),
             starts=i32(B + 1), slots=torch.empty(tokens + 5, dtype=torch.int64, device=DEV),
             positions=i32(tokens + 5), requests=i32(tokens + 5))


def _heads(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def _prepare_prep(case, g, order, s):
    T, hq, hk, D, rot = case["tokens"], case["q_heads"], case["kv_heads"], case["head"], case["rot"]
    src, dt, bs = DTYPES[case["source"]], DTYPES[case["dtype"]], case["block"]
    n_blocks = _blocks(T, bs) + 2
    q = _heads(g, (T, hq, D * (2 if case["gate"] else 1)), src, 3.0)
    slots = torch.randperm(n_blocks * bs, generator=g, device=DEV)[:T]
    if T > 8:
        slots[T // 3] = -1  # a padded place of the batch
    # whole blocks of one head, as the attention reads them; one spare block for the plain form
    caches = [torch.zeros((n_blocks + 1, hk, bs, D), dtype=dt, device=DEV) for _ in range(2)]
    if case["axes"] == 1:
        positions = torch.randint(0, 40000, (1, T), generator=g, device=DEV, dtype=torch.int32)
        axis = [0] * (rot // 2)
    else:  # text advances all three axes, an image's rows and columns the other two
        positions = torch.randint(0, 20000, (3, T), generator=g, device=DEV, dtype=torch.int32)
        axis = [i % 3 for i in range(rot // 2)]
    freq = torch.tensor([10000000.0 ** (-2.0 * i / rot) for i in range(rot // 2)], dtype=torch.float32, device=DEV)
    weights = [_heads(g, (D,), torch.bfloat16, 0.1) if case["norm"] else None for _ in range(2)]
    s.update(q=q[:, :, :D], k=_heads(g, (T, hk, D), src, 2.0), v=_heads(g, (T, hk, D), src), slots=slots,
             positions=positions, axis=axis, axis_dev=_ints(axis, torch.int64), freq=freq, q_norm=weights[0],
             k_norm=weights[1], query=torch.empty((T, hq, D), dtype=dt, device=DEV), pools=caches,
             k_cache=caches[0][:n_blocks].transpose(1, 2), v_cache=caches[1][:n_blocks].transpose(1, 2))


def _prepare_attn(case, g, order, s):
    new, rows = _attn_lengths(case)
    new, rows = [new[i] for i in order], [rows[i] for i in order]
    B, P, D, bs = case["batch"], case["prefix"], case["head"], case["block"]
    hq, hk, dt, T = case["q_heads"], case["kv_heads"], DTYPES[case["dtype"]], sum(new)
    pre, width = _blocks(P, bs), max(_blocks(o, bs) for o in rows)
    held = [_blocks(o, bs) for o in rows]
    n_blocks = pre + sum(held) + 1
    numbers = torch.randperm(n_blocks - 1, generator=g, device=DEV).to(torch.int32)
    tables = torch.full((B, width), -1, dtype=torch.int32, device=DEV)
    at = torch.arange(width, device=DEV)[None, :] < _ints(held, torch.int64)[:, None]
    tables[at] = numbers[pre:pre + sum(held)]
    k = _heads(g, (n_blocks, hk, bs, D), dt)
    v = _heads(g, (n_blocks, hk, bs, D), dt)
    starts = list(itertools.accumulate(new, initial=0))
    s.update(q=_heads(g, (T, hq, D), dt, 1.5), gate=_heads(g, (T, hq, D), dt, 2.0) if case["gate"] else None,
             k_cache=k.transpose(1, 2), v_cache=v.transpose(1, 2), tables=tables,
             lens=_ints([P + o for o in rows]), starts=_ints(starts), prefix_blocks=numbers[:pre].clone(), prefix=P,
             max_new=max(new), width=width, out=torch.empty((T, hq, D), dtype=dt, device=DEV), work=None)


def _prepare_logits(case, g, order, s):
    M, V, L, nb = case["rows"], case["vocab"], case["history"], case["biases"]
    lens = _lengths(case, "history", M, 0, L)
    lens = [lens[i] for i in order]
    # words repeat as in text: small numbers often
    hist = (torch.rand((M, L), generator=g, device=DEV) ** 3 * V).to(torch.int32).clamp_(0, V - 1)
    rnd = lambda lo, hi: lo + (hi - lo) * torch.rand(M, generator=g, device=DEV)  # noqa: E731
    ids = bias = None
    if nb:  # different tokens in a row
        step = max(1, V // nb)
        ids = (torch.arange(nb, device=DEV)[None, :] * step + torch.randint(0, step, (M, 1), generator=g, device=DEV))
        ids = ids.to(torch.int32).contiguous()
        bias = torch.randn((M, nb), generator=g, device=DEV) * 4
    mask = None
    if case["mask"]:
        mask = torch.randint(-2 ** 31, 2 ** 31, (M, _blocks(V, 32)), generator=g, device=DEV, dtype=torch.int64)
        mask = mask.to(torch.int32)
    lens = _ints(lens)
    s.update(logits=torch.randn((M, V), generator=g, device=DEV) * 3, history=hist, lens=lens,
             prompts=(lens * torch.rand(M, generator=g, device=DEV)).to(torch.int32), repetition=rnd(1.0, 1.5),
             presence=rnd(0.0, 1.0), frequency=rnd(0.0, 0.5), ids=ids, bias=bias, mask=mask,
             out=torch.empty((M, V), device=DEV))


# ------------------------------------------------------------------------------ the pass

def run(s):
    if own:
        return {"plan": _own_plan, "prep": _own_prep, "attn": _own_attn, "logits": _own_logits}[s["case"]["op"]](s)
    return {"plan": _plain_plan, "prep": _plain_prep, "attn": _plain_attn, "logits": _plain_logits}[s["case"]["op"]](s)


def _own_plan(s):
    _lib().batch_plan(s["lens"], s["new"], s["tables"], s["pool"], s["free"], s["block"], s["lens_out"],
                      s["free_out"], s["starts"], s["slots"], s["positions"], s["requests"], prefix_len=s["prefix"])
    return (s["lens_out"], s["free_out"], s["starts"], s["slots"], s["positions"], s["requests"], s["tables"],
            s["pool"])


def _plain_plan(s):
    bs, P, T, pool, tables = s["block"], s["prefix"], s["tokens"], s["pool"], s["tables"]
    lens, new, free = s["lens"].long(), s["new"].long(), s["free"].long()
    B, width = tables.shape
    rows = (lens - P).clamp(min=0)
    held = (rows + bs - 1) // bs
    n = new.clamp(min=0)
    back = torch.where(new < 0, held, 0)  # blocks that ended requests give back
    back_end = back.cumsum(0)
    total = (rows + n + bs - 1) // bs
    fits = (n > 0) & (total <= width)
    need = torch.where(fits, total - held, 0)
    need_end, token_end = need.cumsum(0), torch.where(fits, n, 0).cumsum(0)
    have = free + back_end[-1]
    served = fits & (need_end <= have) & (token_end <= T)
    n = torch.where(served, n, 0)
    need = torch.where(served, need, 0)
    need_start = need.cumsum(0) - need
    starts = torch.cat([torch.zeros_like(n[:1]), n.cumsum(0)])
    lens_out = torch.where(served, torch.maximum(lens, torch.full_like(lens, P)) + n, torch.where(new < 0, 0, lens))
    # the pool with what came back on top, and what is taken from its end
    at = torch.arange(pool.numel(), device=pool.device)
    giver = torch.searchsorted(back_end, at - free, right=True).clamp(max=B - 1)
    place = (at - free - (back_end - back)[giver]).clamp(0, width - 1)
    stack = torch.where((at >= free) & (at < have), tables[giver, place], pool)
    left = have - need.sum()
    col = torch.arange(width, device=pool.device)[None, :]
    fresh = (col >= held[:, None]) & (col < (held + need)[:, None])
    taken = stack[(have - 1 - need_start[:, None] - (col - held[:, None])).clamp(0, pool.numel() - 1)]
    tables_out = torch.where(fresh, taken, tables)
    pool_out = torch.where((at >= free) & (at < left), stack, pool)
    token = torch.arange(T, device=pool.device)
    r = torch.searchsorted(starts[1:], token, right=True)
    real = token < starts[-1]
    r = r.clamp(max=B - 1)
    row = rows[r] + token - starts[r]
    slots = tables_out[r, (row // bs).clamp(max=width - 1)].long() * bs + row % bs
    i32 = lambda x: x.to(torch.int32)  # noqa: E731
    return (i32(lens_out), i32(left), i32(starts), torch.where(real, slots, -1), i32(torch.where(real, P + row, -1)),
            i32(torch.where(real, r, -1)), tables_out, pool_out)


def _own_prep(s):
    _lib().paged_prep(s["q"], s["k"], s["v"], s["slots"], s["positions"], s["query"], s["k_cache"], s["v_cache"],
                      inv_freq=s["freq"], axes=s["axis"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS)
    return s["query"], s["k_cache"], s["v_cache"]


def _rotated(x, weight, cos, sin):
    """x f32 [T][heads][D] normalised (weight given) and its first channels rotated."""
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * (1.0 + weight.float())
    half = cos.shape[-1]
    a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)


def _plain_prep(s):
    angle = s["positions"].float()[s["axis_dev"], :].t() * s["freq"]  # [T][rot / 2]
    cos, sin = angle.cos()[:, None, :], angle.sin()[:, None, :]
    slots = s["slots"]
    real = (slots >= 0)[:, None, None]
    query = torch.where(real, _rotated(s["q"].float(), s["q_norm"], cos, sin), 0.0).to(s["query"].dtype)
    rows = _rotated(s["k"].float(), s["k_norm"], cos, sin), s["v"].float()
    kp, vp = s["pools"]
    bs = kp.shape[2]
    at = torch.where(slots >= 0, slots, (kp.shape[0] - 1) * bs)  # padded places go to the spare block
    kp[at // bs, :, at % bs] = rows[0].to(kp.dtype)
    vp[at // bs, :, at % bs] = rows[1].to(vp.dtype)
    return query, s["k_cache"], s["v_cache"]


def _own_attn(s):
    Y = _lib()
    if s["work"] is None:
        n = Y.prefix_attention_work_bytes(s["q"].shape[0], s["tables"].shape[0], s["max_new"], s["q"].shape[1],
                                          s["k_cache"].shape[2], s["q"].shape[2])
        s["work"] = torch.empty(n, dtype=torch.uint8, device=DEV)
    Y.prefix_attention(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["lens"], s["starts"], s["max_new"],
                       s["work"], s["out"], prefix_blocks=s["prefix_blocks"], prefix_len=s["prefix"],
                       gate=s["gate"])
    return s["out"]


def _plain_attn(s):
    q, kc, vc, P, n_max = s["q"].float(), s["k_cache"], s["v_cache"], s["prefix"], s["max_new"]
    (T, hq, D), hk, bs = q.shape, kc.shape[2], kc.shape[1]
    G, B = hq // hk, s["tables"].shape[0]
    starts, lens = s["starts"].long(), s["lens"].long()
    n = starts[1:] - starts[:-1]
    # rows padded to n_max a request: [B][hk][n_max * G][D]
    j = torch.arange(n_max, device=q.device)
    token = (starts[:-1, None] + j[None, :]).clamp(max=T - 1)
    limit = (lens[:, None] - n[:, None] + j[None, :] + 1).clamp(min=0)  # rows of the sequence that a token sees
    qp = q[token].view(B, n_max, hk, G, D).permute(0, 2, 1, 3, 4).reshape(B, hk, n_max * G, D)
    flat = lambda c, t: c[t.clamp(min=0).long()].flatten(-4, -3).float()  # noqa: E731  blocks -> rows [..][hk][D]
    kp, vp = (flat(c, s["prefix_blocks"])[:P].transpose(0, 1) for c in (kc, vc))  # [hk][P][D]
    ko, vo = (flat(c, s["tables"]).transpose(1, 2) for c in (kc, vc))  # [B][hk][width * bs][D]
    rows = torch.arange(ko.shape[2], device=q.device)
    vo = torch.where((P + rows < lens[:, None])[:, None, :, None], vo, 0.0)
    limit = limit[:, None, :, None, None]  # against scores [B][hk][n_max][G][rows]
    scale = 1.0 / math.sqrt(D)
    sp = torch.matmul(qp, kp.transpose(-1, -2)[None]).mul_(scale).view(B, hk, n_max, G, P)
    so = torch.matmul(qp, ko.transpose(-1, -2)).mul_(scale).view(B, hk, n_max, G, -1)
    sp.masked_fill_(torch.arange(P, device=q.device) >= limit, -math.inf)
    so.masked_fill_(P + rows >= limit, -math.inf)
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


def _own_logits(s):
    _lib().logits_adjust(s["logits"], s["out"], history=s["history"], history_lens=s["lens"],
                         prompt_lens=s["prompts"], repetition=s["repetition"], presence=s["presence"],
                         frequency=s["frequency"], bias_ids=s["ids"], bias=s["bias"], mask=s["mask"])
    return s["out"]


def _plain_logits(s):
    x = s["logits"]
    M, V = x.shape
    hist = s["history"].long()
    at = torch.arange(hist.shape[1], device=x.device)[None, :]
    real = at < s["lens"][:, None]
    zero = torch.zeros((M, V), dtype=torch.int32, device=x.device)
    seen = zero.scatter_add(1, hist, real.int())
    said = zero.scatter_add(1, hist, (real & (at >= s["prompts"][:, None])).int())
    rep = s["repetition"][:, None]
    x = torch.where(seen > 0, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"][:, None] * said.float() - s["presence"][:, None] * (said > 0).float()
    if s["ids"] is not None:
        x = x.scatter_add(1, s["ids"].long(), s["bias"])
    if s["mask"] is not None:
        t = torch.arange(V, device=x.device)
        x = torch.where((s["mask"][:, t >> 5] >> (t & 31)) & 1 == 1, x, -math.inf)
    return x


# ------------------------------------------------------------- the definitions in 64 bits

def exact(case, seed):
    f64 = torch.float64

    def heads_and_rows(s):
        half = s["freq"].numel()
        # the angle is the 32-bit product of position and frequency, as the decode path's rotation
        angle = torch.stack([s["positions"][a].to(torch.float32) * s["freq"][i] for i, a in enumerate(s["axis"])], 1)
        turn = torch.polar(torch.ones_like(angle, dtype=f64), angle.to(f64))[:, None, :]

        def heads(x, w):
            x = x.to(f64)
            if w is not None:
                x = x / ((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * (1 + w.to(f64))
            z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * turn
            return torch.cat((z.real, z.imag, x[..., 2 * half:]), -1)

        keep = s["slots"] >= 0
        query = heads(s["q"], s["q_norm"])
        query[~keep] = 0
        out = [query]
        for rows, cache in ((heads(s["k"], s["k_norm"]), s["k_cache"]), (s["v"].to(f64), s["v_cache"])):
            whole = torch.zeros(cache.shape, dtype=f64, device=DEV)
            bs = cache.shape[1]
            at = s["slots"][keep]
            whole[at // bs, at % bs] = rows[keep]
            out.append(whole)
        return tuple(out)

    def attention(s):
        P, T = s["prefix"], s["q"].shape[0]
        hq, D, hk, bs = s["q"].shape[1], s["q"].shape[2], s["k_cache"].shape[2], s["k_cache"].shape[1]
        G = hq // hk
        lens, starts = s["lens"].tolist(), s["starts"].tolist()
        kp = s["k_cache"][s["prefix_blocks"].long()].reshape(-1, hk, D)[:P].to(f64)
        vp = s["v_cache"][s["prefix_blocks"].long()].reshape(-1, hk, D)[:P].to(f64)
        out = torch.zeros((T, hq, D), dtype=f64, device=DEV)
        for b, length in enumerate(lens):
            t0, t1 = starts[b], starts[b + 1]
            ids = s["tables"][b, :_blocks(length - P, bs)].long()
            k = torch.cat([kp, s["k_cache"][ids].reshape(-1, hk, D)[:length - P].to(f64)])
            v = torch.cat([vp, s["v_cache"][ids].reshape(-1, hk, D)[:length - P].to(f64)])
            at = torch.arange(length, device=DEV)
            hidden = at[None, :] > at[length - (t1 - t0):, None]
            for h in range(hk):
                q = s["q"][t0:t1, h * G:(h + 1) * G].to(f64)  # [n][G][D]
                w = torch.einsum("ngd,ld->gnl", q, k[:, h]) / math.sqrt(D)
                w = torch.softmax(w.masked_fill(hidden[None], -math.inf), -1)
                out[t0:t1, h * G:(h + 1) * G] = torch.einsum("gnl,ld->ngd", w, v[:, h])
        if s["gate"] is not None:
            out = out / (1 + torch.exp(-s["gate"].to(f64)))
        return out

    def logits(s):
        x = s["logits"].to(f64)
        M, V = x.shape
        lens, prompts = s["lens"].tolist(), s["prompts"].tolist()
        for m in range(M):
            seen = torch.bincount(s["history"][m, :lens[m]].long(), minlength=V)
            said = torch.bincount(s["history"][m, prompts[m]:lens[m]].long(), minlength=V)
            rep = s["repetition"][m].to(f64)
            row = x[m]
            row = torch.where(seen > 0, row * torch.where(row > 0, 1 / rep, rep), row)
            row = row - said * s["frequency"][m].to(f64) - said.clamp(max=1) * s["presence"][m].to(f64)
            if s["ids"] is not None:
                row[s["ids"][m].long()] += s["bias"][m].to(f64)
            if s["mask"] is not None:
                bits = torch.stack([(s["mask"][m] >> b) & 1 for b in range(32)], 1).reshape(-1)[:V]
                row[bits == 0] = -math.inf
            x[m] = row
        return x

    if case["op"] == "plan":
        return None  # whole numbers: held equal
    return {"prep": heads_and_rows, "attn": attention, "logits": logits}[case["op"]](prepare(case, seed))
