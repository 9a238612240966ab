"""Refusals of the operators for drafted trees, forked requests and log probabilities: bad shapes, types, strides and
alignment come back as EINVAL with a message before any device work (fake, never dereferenced pointers; no GPU)."""
import ctypes as C
import os
import shutil
import struct
import subprocess

import pytest

P = 4096  # stands for a device pointer; 16-byte aligned

TREE_PLAN = dict(parents=P, requests=P, starts=P, lens=P, mask=P, stride=2, positions=P, tokens=5, batch=2, words=2)
ATTENTION = dict(q=P, q_row=512, q_head=128, gate=None, gate_row=0, gate_head=0, k=P, v=P, block=4096, token=128,
                 head_stride=2048, prefix_blocks=P, tables=P, stride=2, lens=P, starts=P, work=P, work_bytes=1 << 30,
                 out=P, n_blocks=3, block_size=16, prefix=20, width=2, batch=2, tokens=3, max_new=2, n_qh=4, n_kvh=2,
                 head=128, dtype=2, gate_dtype=2, scale=0.1, mask=P, mask_stride=1, words=1)
TREE_ACCEPT = dict(tokens=P, parents=P, choice=P, starts=P, lens=P, path=P, stride=4, accepted=P, lens_out=P, next=P,
                   batch=2, n_tokens=5, width=4)
BATCH_EDIT = dict(lens=P, keep=P, source=P, tables=P, stride=4, tables_out=2 * P, out_stride=4, pool=P, free=P,
                  lens_out=2 * P, free_out=2 * P, copies=P, copies_stride=9, n_copies=P, batch=2, block=16, prefix=0,
                  width=4, capacity=9, max_copies=9)
LOGPROBS = dict(logits=P, stride=100, tokens=P, token_stride=3, logprobs=P, entropy=None, tops=P, ids=P, rows=2,
                vocab=100, n_tokens=3, n_top=5)


def caches(*pointers):
    a = (C.c_void_p * len(pointers))(*pointers)
    return a, C.addressof(a)


KEEP, AT = caches(P, 2 * P)
COPY = dict(caches=AT, block=4096, token=128, head_stride=2048, copies=P, copies_stride=9, count=None, n=2, n_blocks=3,
            block_size=16, n_kvh=2, head=128, max_copies=9)
COMPACT = dict(caches=AT, block=4096, token=128, head_stride=2048, tables=P, stride=4, lens=P, starts=P, path=P,
               path_stride=5, n=2, n_blocks=3, block_size=16, n_kvh=2, head=128, batch=2, width=4, prefix=0,
               path_width=5)


def refused(name, good, bad):
    import yskn_b200 as Y
    fn, args_of = getattr(Y.lib(), "yskn_b200_" + name), Y.ARGS[name]
    assert fn(None, None) == Y.EINVAL and name in Y.last_error()
    for i, change in enumerate(bad):
        args = dict(good, **change)
        assert list(args) == list(good)
        assert fn(args_of.pack(*(0 if v is None else v for v in args.values())), None) == Y.EINVAL, (name, i, change)
        assert name in Y.last_error()


def test_tree_plan():
    refused("tree_plan", TREE_PLAN,
            [{k: None} for k in ("parents", "requests", "starts", "lens", "mask", "positions")] +
            [dict(tokens=0), dict(tokens=-1), dict(tokens=2 ** 30 + 1), dict(batch=0), dict(words=0), dict(words=33),
             dict(stride=1)])


def test_tree_attention():
    import yskn_b200 as Y
    refused("tree_attention", ATTENTION,
            [{k: None} for k in ("q", "k", "v", "prefix_blocks", "tables", "lens", "starts", "work", "out", "mask")] +
            [{k: P + 8} for k in ("q", "gate", "k", "v", "work", "out")] +
            [dict(words=0), dict(mask_stride=0), dict(head=96), dict(dtype=0), dict(tokens=0), dict(batch=0),
             dict(max_new=0), dict(n_kvh=3), dict(n_qh=258), dict(prefix=-1), dict(stride=1), dict(n_blocks=0),
             dict(block_size=48), dict(q_row=516), dict(gate=P, gate_dtype=1),
             dict(work_bytes=Y.prefix_attention_work_bytes(3, 2, 2, 4, 2, 128) - 1)])


def test_tree_accept():
    refused("tree_accept", TREE_ACCEPT,
            [{k: None} for k in ("tokens", "parents", "choice", "starts", "lens", "path", "accepted", "lens_out",
                                 "next")] +
            [dict(batch=0), dict(n_tokens=0), dict(n_tokens=2 ** 30 + 1), dict(batch=2 ** 30 + 1), dict(width=0),
             dict(stride=3)])


def test_batch_edit():
    refused("batch_edit", BATCH_EDIT,
            [{k: None} for k in ("lens", "keep", "tables", "tables_out", "pool", "free", "lens_out", "free_out",
                                 "copies", "n_copies")] +
            [dict(batch=0), dict(batch=4097), dict(block=0), dict(prefix=-1), dict(width=0), dict(stride=3),
             dict(out_stride=3), dict(capacity=0), dict(max_copies=0), dict(copies_stride=8), dict(lens_out=P),
             dict(free_out=P), dict(tables_out=P)])


def test_cache_moves():
    null, none = caches(P, 0)
    odd, crooked = caches(P, P + 8)
    shapes = [dict(caches=None), dict(caches=none), dict(caches=crooked), dict(n=0), dict(n=257), dict(n_blocks=0),
              dict(block_size=0), dict(n_kvh=0), dict(head=96), dict(head=8), dict(block=4), dict(token=4),
              dict(head_stride=4)]
    refused("cache_copy", COPY, shapes + [dict(copies=None), dict(max_copies=0), dict(copies_stride=8),
                                          dict(block_size=2 ** 31 - 1, n_kvh=2 ** 20)])
    refused("cache_compact", COMPACT,
            shapes + [{k: None} for k in ("tables", "lens", "starts", "path")] +
            [dict(batch=0), dict(width=0), dict(prefix=-1), dict(path_width=0), dict(stride=3), dict(path_stride=4)])
    assert null and odd


def test_token_logprobs():
    refused("token_logprobs", LOGPROBS,
            [{k: None} for k in ("logits", "tokens", "logprobs", "tops", "ids")] +
            [dict(rows=0), dict(rows=2 ** 31 - 1), dict(vocab=0), dict(vocab=2 ** 31 - 1), dict(stride=99),
             dict(token_stride=2), dict(n_tokens=-1), dict(n_top=-1), dict(n_top=33)])


@pytest.mark.parametrize("name,last", [("tree_plan", "mask_words"), ("tree_attention", "mask_words"),
                                       ("tree_accept", "path_width"), ("batch_edit", "max_copies"),
                                       ("cache_copy", "max_copies"), ("cache_compact", "path_width"),
                                       ("token_logprobs", "n_top")])
def test_packed_arguments_are_the_whole_struct(tmp_path, name, last):
    """The library copies the struct whole: its padding at the end has to be there too."""
    import yskn_b200 as Y
    from conftest import ROOT
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    src, exe = tmp_path / "s.c", tmp_path / "s"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "yskn_b200.h"\n'
                   'int main(void) { printf("%%zu %%zu", '
                   'sizeof(yskn_b200_%s_args), offsetof(yskn_b200_%s_args, %s)); return 0; }' % (name, name, last))
    subprocess.run([cc, "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    size, at = map(int, subprocess.run([str(exe)], capture_output=True, check=True).stdout.split())
    assert Y.ARGS[name].size == size
    whole = Y.ARGS[name].format
    assert whole.endswith("0P") and struct.calcsize(whole[:-2]) - 4 == at


def test_the_binding_refuses_what_the_c_entry_cannot_see():
    """Types, shapes, strides and devices (CPU tensors: nothing is launched)."""
    import torch
    import yskn_b200 as Y
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    f32 = lambda *s: torch.zeros(s)  # noqa: E731
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16)  # noqa: E731
    every_second = lambda t: torch.stack([t, t], -1)[..., 0]  # noqa: E731

    class Stream:
        cuda_stream = 0

    def no(fn, good, what=None, **change):
        with pytest.raises(Y.YsknError, match="^" + (what or fn.__name__) + ": ") as e:
            fn(stream=Stream, **dict(good, **change))
        assert e.value.code == Y.EINVAL

    def arrays(fn, good, names):
        for k in names:
            no(fn, good, **{k: good[k].double()})
            if good[k].dim() == 1 and good[k].numel() > 1:
                no(fn, good, **{k: every_second(good[k])})
                no(fn, good, **{k: torch.cat([good[k], good[k]])})

    plan = dict(parents=i32(5), requests=i32(5), starts=i32(3), lens=i32(2), mask=i32(5, 2), positions=i32(5))
    arrays(Y.tree_plan, plan, plan)
    no(Y.tree_plan, plan)  # not on a GPU
    no(Y.tree_plan, plan, mask=i32(4, 2))
    no(Y.tree_plan, plan, mask=i32(2, 5).t())
    acc = dict(tokens=i32(5), parents=i32(5), choice=i32(5), starts=i32(3), lens=i32(2), path=i32(2, 3),
               accepted=i32(2), lens_out=i32(2), next_token=i32(2))
    arrays(Y.tree_accept, acc, acc)
    no(Y.tree_accept, acc)
    no(Y.tree_accept, acc, path=i32(3, 2).t())
    c = bf(5, 16, 2, 64)
    att = dict(q=bf(3, 4, 64), k_cache=c, v_cache=c, block_tables=i32(2, 3), lens=i32(2), starts=i32(3), max_new=2,
               mask=i32(3, 1), work=torch.zeros(1 << 24, dtype=torch.uint8), out=bf(3, 4, 64))
    arrays(Y.tree_attention, att, ("lens", "starts", "mask", "q", "out", "k_cache", "block_tables"))
    no(Y.tree_attention, att)
    no(Y.tree_attention, att, mask=i32(2, 1))
    edit = dict(lens=i32(2), keep=i32(2), block_tables=i32(2, 3), pool=i32(4), free_count=i32(1), block_size=16,
                lens_out=i32(2), free_out=i32(1), source=i32(2), tables_out=i32(2, 3), copies=i32(3, 6),
                n_copies=i32(1))
    arrays(Y.batch_edit, edit, ("lens", "keep", "block_tables", "free_count", "lens_out", "free_out", "source",
                                "tables_out", "copies", "n_copies"))
    no(Y.batch_edit, edit)
    for k in ("tables_out", "copies", "n_copies"):
        no(Y.batch_edit, edit, **{k: None})
    no(Y.batch_edit, edit, copies=i32(6, 3).t())
    no(Y.batch_edit, edit, tables_out=i32(2, 4))
    for bad in ([], [c, c.half()], [c, bf(5, 16, 2, 128)], [c.float()], [c, bf(5, 2, 16, 64).transpose(1, 2)],
                [bf(5, 16, 64, 2).transpose(2, 3)]):
        with pytest.raises(Y.YsknError, match="^CacheSet: "):
            Y.CacheSet(bad)
    both = Y.CacheSet([c, c])
    copy = dict(caches=both, copies=i32(3, 6), count=i32(1))
    arrays(Y.cache_copy, copy, ("copies", "count"))
    no(Y.cache_copy, copy)
    no(Y.cache_copy, copy, copies=i32(2, 6))
    pack = dict(caches=both, block_tables=i32(2, 3), lens=i32(2), starts=i32(3), path=i32(2, 4))
    arrays(Y.cache_compact, pack, ("block_tables", "lens", "starts", "path"))
    no(Y.cache_compact, pack)
    no(Y.cache_compact, pack, path=i32(1, 4))
    lp = dict(logits=f32(2, 50), tokens=i32(2, 3), logprobs=f32(2, 3), entropy=f32(2), top_logprobs=f32(2, 4),
              top_ids=i32(2, 4))
    arrays(Y.token_logprobs, lp, lp)
    no(Y.token_logprobs, lp)
    for k in ("tokens", "logprobs", "top_logprobs", "top_ids"):
        no(Y.token_logprobs, lp, **{k: None})
    no(Y.token_logprobs, lp, logits=f32(50, 2).t())
    no(Y.token_logprobs, lp, logprobs=f32(3, 2).t())


def test_batch_edit_writes_lengths_to_an_array_of_their_own():
    refused("batch_edit", BATCH_EDIT, [dict(keep=2 * P), dict(source=2 * P), dict(keep=2 * P, source=None)])
