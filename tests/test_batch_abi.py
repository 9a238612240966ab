"""Refusals of the batch operators: bad shapes, types, strides and alignment come back as EINVAL
with a message before any device work (fake, never dereferenced pointers; no GPU needed)."""
import pytest

P = 4096  # stands for a device pointer; 16-byte aligned


def _check(name, good, bad):
    import yskn_b200 as Y
    fn, args_of = getattr(Y.lib(), name), Y.ARGS[name.replace("yskn_b200_", "")]
    assert fn(None, None) == Y.EINVAL
    for i, change in enumerate(bad):
        args = dict(good, **change)
        assert list(args) == list(good)
        packed = args_of.pack(*(0 if v is None else v for v in args.values()))
        assert fn(packed, None) == Y.EINVAL, (name, i, change)
        assert name.replace("yskn_b200_", "") in Y.last_error()


def test_batch_plan():
    good = dict(lens=P, new=P, tables=P, stride=4, pool=P, free=P, lens_out=2 * P, free_out=2 * P, starts=P, slots=P,
                positions=P, requests=P, batch=2, block=16, prefix=0, width=4, capacity=9, tokens=5)
    _check("yskn_b200_batch_plan", good,
           [{k: None} for k in ("lens", "new", "tables", "pool", "free", "lens_out", "free_out", "starts", "slots",
                                "positions", "requests")] +
           [dict(batch=0), dict(batch=4097), dict(block=0), dict(prefix=-1), dict(width=0), dict(stride=3),
            dict(capacity=0), dict(tokens=-1), dict(lens_out=P), dict(free_out=P)])


def test_paged_prep():
    good = dict(q=P, k=P, v=P, q_row=512, q_head=128, k_row=256, k_head=128, v_row=256, v_head=128, slots=P,
                positions=P, position_stride=4, freq=P, q_norm=P, k_norm=P, query=P, k_cache=P, v_cache=P, block=4096,
                token=128, head_stride=2048, tokens=4, n_qh=4, n_kvh=2, head=128, rot=64, n_axes=3, n_blocks=3,
                block_size=16, source=0, dtype=2, eps=1e-6, axes=bytes(32))
    _check("yskn_b200_paged_prep", good,
           [{k: None} for k in ("q", "k", "v", "slots", "positions", "freq", "query", "k_cache", "v_cache")] +
           [{k: P + 8} for k in ("q", "k", "v", "query", "k_cache", "v_cache", "q_norm", "k_norm")] +
           [dict(head=96), dict(head=512), dict(dtype=0), dict(dtype=3), dict(source=1), dict(source=7),
            dict(tokens=0), dict(n_qh=0), dict(n_kvh=0), dict(rot=-16), dict(rot=144), dict(rot=24),
            dict(axes=bytes([3]) * 32, n_axes=4), dict(axes=bytes([1]) * 32, n_axes=1), dict(q_row=514), dict(k_head=130), dict(block=4), dict(token=4),
            dict(head_stride=4), dict(n_blocks=0), dict(block_size=0)])


def test_prefix_attention():
    import yskn_b200 as Y
    good = dict(q=P, q_row=512, q_head=128, gate=None, gate_row=0, gate_head=0, k=P, v=P, block=4096, token=128,
                head_stride=2048, prefix_blocks=P, tables=P, stride=2, lens=P, starts=P, work=P, work_bytes=1 << 30,
                out=P, n_blocks=3, block_size=16, prefix=20, width=2, batch=2, tokens=3, max_new=2, n_qh=4, n_kvh=2,
                head=128, dtype=2, gate_dtype=2, scale=0.1)
    _check("yskn_b200_prefix_attention", good,
           [{k: None} for k in ("q", "k", "v", "prefix_blocks", "tables", "lens", "starts", "work", "out")] +
           [{k: P + 8} for k in ("q", "gate", "k", "v", "work", "out")] +
           [dict(head=96), dict(dtype=0), dict(dtype=3), dict(tokens=0), dict(batch=0), dict(max_new=0), dict(n_kvh=0),
            dict(n_kvh=3), dict(n_qh=258), dict(prefix=-1), dict(width=0), dict(stride=1), dict(n_blocks=0),
            dict(block_size=8), dict(block_size=48), dict(block_size=256), dict(q_row=516), dict(q_head=4),
            dict(block=4), dict(token=4), dict(head_stride=4), dict(gate=P, gate_row=4),
            dict(gate=P, gate_dtype=1), dict(gate=P, gate_dtype=0, gate_row=2),
            dict(work_bytes=Y.prefix_attention_work_bytes(3, 2, 2, 4, 2, 128) - 1)])
    L = Y.lib()
    assert L.yskn_b200_prefix_attention_work_bytes(3, 2, 2, 4, 2, 128) > 0
    for args in [(0, 2, 2, 4, 2, 128), (3, 0, 2, 4, 2, 128), (3, 2, 0, 4, 2, 128), (3, 2, 2, 5, 2, 128),
                 (3, 2, 2, 4, 0, 128), (3, 2, 2, 4, 2, 100)]:
        assert L.yskn_b200_prefix_attention_work_bytes(*args) == -1
    with pytest.raises(Y.YsknError):
        Y.prefix_attention_work_bytes(0, 2, 2, 4, 2, 128)


def test_logits_adjust():
    good = dict(logits=P, logits_stride=100, history=P, history_stride=10, lens=P, prompts=None, rep=P, pres=None,
                freq=None, ids=P, bias=P, mask=P, mask_stride=4, out=P, out_stride=100, rows=2, vocab=100, width=10,
                n_bias=3)
    _check("yskn_b200_logits_adjust", good,
           [{k: None} for k in ("logits", "lens", "ids", "bias", "out")] +
           [dict(rows=0), dict(rows=65536), dict(vocab=0), dict(vocab=2 ** 31 - 1), dict(logits_stride=99),
            dict(out_stride=99), dict(width=-1), dict(history_stride=9), dict(history=None), dict(n_bias=-1),
            dict(mask_stride=3)])


def test_tensor_checks_of_the_binding():
    """Types, shapes and strides that the C entry cannot see (CPU tensors: nothing is launched)."""
    import torch
    import yskn_b200 as Y
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    i64 = lambda *s: torch.zeros(s, dtype=torch.int64)  # noqa: E731
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16)  # noqa: E731
    f32 = lambda *s: torch.zeros(s)  # noqa: E731

    class Stream:  # the legacy default stream; what the C entry refuses never gets to it
        cuda_stream = 0

    def refused(fn, *a, **k):
        with pytest.raises(Y.YsknError) as e:
            fn(*a, stream=Stream, **k)
        assert e.value.code == Y.EINVAL

    plan = lambda **k: [dict(dict(lens=i32(2), new=i32(2), tables=i32(2, 3), pool=i32(4), free=i32(1), bs=16,  # noqa: E731
                                  lo=i32(2), fo=i32(1), st=i32(3), sl=i64(4), po=i32(4), rq=i32(4)), **k)[x]
                        for x in ("lens", "new", "tables", "pool", "free", "bs", "lo", "fo", "st", "sl", "po", "rq")]
    refused(Y.batch_plan, *plan(lens=i64(2)))
    refused(Y.batch_plan, *plan(st=i32(2)))
    refused(Y.batch_plan, *plan(sl=i32(4)))
    refused(Y.batch_plan, *plan(po=i32(3)))
    refused(Y.batch_plan, *plan(tables=i32(3, 2).t()))
    q, k, c = f32(3, 4, 64), f32(3, 2, 64), bf(5, 16, 2, 64)
    refused(Y.paged_prep, q, k, k, i64(2), i32(3), bf(3, 4, 64), c, c)
    refused(Y.paged_prep, q, k, k, i64(3), i32(3), bf(3, 4, 128), c, c)
    refused(Y.paged_prep, q, k, k, i64(3), i32(3), bf(3, 4, 64), c, c.to(torch.float16))
    refused(Y.paged_prep, q, k, k, i64(3), i32(3), bf(3, 4, 64), c, bf(5, 2, 16, 64).transpose(1, 2))
    refused(Y.paged_prep, q, k, k, i64(3), i32(3), bf(3, 4, 64), c, c, inv_freq=f32(16), axes=[1] * 16)
    refused(Y.paged_prep, q, k, k, i64(3), i32(3), bf(3, 4, 64), c, c, inv_freq=f32(16), axes=[0] * 15)
    refused(Y.paged_prep, q, k, k, i64(3), i64(3), bf(3, 4, 64), c, c, inv_freq=f32(16))
    qa, work = bf(3, 4, 64), torch.zeros(1 << 24, dtype=torch.uint8)
    att = lambda **k: Y.prefix_attention(*[dict(dict(q=qa, kc=c, vc=c, tb=i32(2, 3), ln=i32(2), st=i32(3), mn=2,  # noqa: E731
                                                     wk=work, out=bf(3, 4, 64)), **k)[x]
                                           for x in ("q", "kc", "vc", "tb", "ln", "st", "mn", "wk", "out")],
                                         **{x: y for x, y in k.items() if x in ("gate", "prefix_blocks", "prefix_len", "stream")})
    refused(att, q=qa.to(torch.float16))
    refused(att, st=i32(2))
    refused(att, tb=i64(2, 3))
    refused(att, wk=work[:1])
    refused(att, gate=bf(3, 4, 32))
    refused(att, prefix_len=17, prefix_blocks=i32(1))
    refused(att, prefix_len=1)
    x = f32(2, 50)
    refused(Y.logits_adjust, x, bf(2, 50))
    refused(Y.logits_adjust, x, x, history=i64(2, 4), history_lens=i32(2))
    refused(Y.logits_adjust, x, x, bias=f32(2, 3))
    refused(Y.logits_adjust, x, x, bias=f32(2, 3), bias_ids=i32(2, 4))
    refused(Y.logits_adjust, x, x, mask=i32(1, 2))
    refused(Y.logits_adjust, f32(50, 2).t(), x)


@pytest.mark.parametrize("name,last", [("batch_plan", "max_tokens"), ("paged_prep", "axes"),
                                       ("prefix_attention", "scale"), ("logits_adjust", "n_bias")])
def test_packed_arguments_are_the_whole_struct(tmp_path, name, last):
    """The library copies the struct whole: its padding at the end has to be there too."""
    import os
    import shutil
    import struct
    import subprocess
    import yskn_b200 as Y
    from conftest import ROOT
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    src, exe = tmp_path / "s.c", tmp_path / "s"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "yskn_b200.h"\nint main(void) { printf("%%zu %%zu", '
                   'sizeof(yskn_b200_%s_args), offsetof(yskn_b200_%s_args, %s)); return 0; }' % (name, name, last))
    subprocess.run([cc, "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    size, at = map(int, subprocess.run([str(exe)], capture_output=True, check=True).stdout.split())
    assert Y.ARGS[name].size == size
    unpadded = Y.ARGS[name].format.replace("0P", "")
    assert struct.calcsize(unpadded) - (128 if last == "axes" else 4) == at


def test_arrays_that_the_library_reads_by_address_alone():
    """Types, lengths and strides of the arrays whose layout the C entry takes for granted."""
    import torch
    import yskn_b200 as Y
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    i64 = lambda *s: torch.zeros(s, dtype=torch.int64)  # noqa: E731
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16)  # noqa: E731
    f32 = lambda *s: torch.zeros(s)  # noqa: E731
    every_second = lambda t: torch.stack([t, t], -1)[..., 0]  # noqa: E731

    class Stream:
        cuda_stream = 0

    def refused(what, fn, good, **change):
        args = dict(good, **change)
        with pytest.raises(Y.YsknError, match=what) as e:
            fn(stream=Stream, **args)
        assert e.value.code == Y.EINVAL

    plan = dict(lens=i32(2), new_lens=i32(2), block_tables=i32(2, 3), pool=i32(4), free_count=i32(1), block_size=16,
                lens_out=i32(2), free_out=i32(1), starts=i32(3), slots=i64(4), positions=i32(4), requests=i32(4))
    for k, v in plan.items():
        if k not in ("block_tables", "block_size"):
            if v.numel() > 1:
                refused("^batch_plan: ", Y.batch_plan, plan, **{k: every_second(v)})
            refused("^batch_plan: ", Y.batch_plan, plan, **{k: v.to(torch.float64 if k == "slots" else torch.float32)})
    refused("^batch_plan: ", Y.batch_plan, plan, free_count=i32(0))

    c = bf(5, 16, 2, 64)
    prep = dict(q=f32(3, 4, 64), k=f32(3, 2, 64), v=f32(3, 2, 64), slots=i64(3), positions=i32(3), query=bf(3, 4, 64),
                k_cache=c, v_cache=c, inv_freq=f32(16), q_norm=bf(64), k_norm=bf(64))
    refused("slots", Y.paged_prep, prep, slots=f32(3).double())
    refused("slots", Y.paged_prep, prep, slots=every_second(i64(3)))
    for bad in (f32(64), bf(32), bf(128), every_second(bf(64)), torch.zeros(64, dtype=torch.float16)):
        refused("norms", Y.paged_prep, prep, q_norm=bad)
        refused("norms", Y.paged_prep, prep, k_norm=bad)
    for bad in (f32(16).double(), bf(16), every_second(f32(16))):
        refused("frequency|f32", Y.paged_prep, prep, inv_freq=bad)

    att = dict(q=bf(3, 4, 64), k_cache=c, v_cache=c, block_tables=i32(2, 3), lens=i32(2), starts=i32(3), max_new=2,
               work=torch.zeros(1 << 24, dtype=torch.uint8), out=bf(3, 4, 64), prefix_blocks=i32(2), prefix_len=20)
    for k in ("lens", "starts", "prefix_blocks", "work"):
        refused("prefix_attention: dense", Y.prefix_attention, att, **{k: every_second(att[k])})

    adjust = dict(logits=f32(2, 50), out=f32(2, 50), history=i32(2, 4), history_lens=i32(2), prompt_lens=i32(2),
                  repetition=f32(2), presence=f32(2), frequency=f32(2))
    for k in ("history_lens", "prompt_lens", "repetition", "presence", "frequency"):
        refused("logits_adjust: a dense", Y.logits_adjust, adjust, **{k: every_second(adjust[k])})
        refused("logits_adjust: a dense", Y.logits_adjust, adjust, **{k: adjust[k].double()})


def test_work_bytes_without_a_bound_on_the_new_tokens():
    """A request has at most all of the call's tokens: a larger max_new says no more than that."""
    import yskn_b200 as Y
    for G in (1, 2, 4, 6, 8, 16):
        for tokens in (1, 3, 200):
            n = Y.prefix_attention_work_bytes(tokens, 5, tokens, 4 * G, 4, 256)
            for max_new in (tokens + 1, 357913942, 2 ** 30, 2 ** 31 - 1):
                assert Y.prefix_attention_work_bytes(tokens, 5, max_new, 4 * G, 4, 256) == n


def test_the_largest_steps_work_bytes_serve_every_smaller_one():
    import yskn_b200 as Y
    sizes = (1, 2, 3, 4, 8, 16, 41, 64, 300)
    for G in (1, 2, 3, 6, 8, 9):
        for head in (64, 256):
            need = lambda *a: Y.prefix_attention_work_bytes(*a, 4 * G, 4, head)  # noqa: E731
            for T in sizes:
                for B in (1, 7, 64):
                    for n in sizes:
                        most = need(T, B, n)
                        for less in ((max(1, T // 2), B, n), (T, max(1, B // 3), n), (T, B, max(1, n // 2)), (T, B, 1),
                                     (1, 1, 1)):
                            assert need(*less) <= most, (G, head, (T, B, n), less)


def test_plan_of_more_tokens_than_its_places_count():
    """Places of tokens are 32-bit numbers on the device, those that a CTA rounds up to among them."""
    good = dict(lens=P, new=P, tables=P, stride=4, pool=P, free=P, lens_out=2 * P, free_out=2 * P, starts=P, slots=P,
                positions=P, requests=P, batch=2, block=16, prefix=0, width=4, capacity=9, tokens=5)
    _check("yskn_b200_batch_plan", good, [dict(tokens=2 ** 30 + 1), dict(tokens=2 ** 31 - 1)])
