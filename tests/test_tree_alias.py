"""Outputs of the operators for drafted trees and forked requests that would meet what other CTAs or warps still read:
refused with EINVAL and a message before any device work (fake, never dereferenced pointers; no GPU)."""
from test_tree_abi import BATCH_EDIT, P, TREE_ACCEPT, TREE_PLAN


def apart(good, **change):
    """The arguments with an address of its own, a megabyte from the next, for each pointer."""
    at = iter(range(1 << 24, 1 << 30, 1 << 20))
    args = {k: next(at) if v in (P, 2 * P) else v for k, v in good.items()}
    return dict(args, **{k: args[v] if isinstance(v, str) else args[v[0]] + v[1] for k, v in change.items()})


def test_batch_edit_refuses_outputs_that_meet_what_every_cta_reads():
    import yskn_b200 as Y
    fn, args_of = Y.lib().yskn_b200_batch_edit, Y.ARGS["batch_edit"]
    for change in (dict(n_copies="free"), dict(n_copies="free_out"), dict(n_copies=("lens", 4)), dict(n_copies="keep"),
                   dict(free_out=("lens", 4)), dict(free_out="n_copies"), dict(free_out=("source", 4)),
                   dict(free_out=("lens_out", 4)), dict(lens_out=("lens", 4)), dict(lens_out=("keep", -4)),
                   dict(lens_out=("source", 4)), dict(lens_out="free"), dict(pool=("lens", -4)), dict(free=("pool", 32)),
                   dict(lens_out=("pool", 32)), dict(n_copies="pool")):
        assert fn(args_of.pack(*apart(BATCH_EDIT, **change).values()), None) == Y.EINVAL, change
        assert "arrays of their own" in Y.last_error(), change


def passes(fn, args):
    """Not refused: the call goes on to the launch, which no machine without a GPU can do."""
    import torch
    import yskn_b200 as Y
    return torch.cuda.is_available() or fn(args, None) not in (0, Y.EINVAL)


def test_tree_plan_refuses_outputs_that_meet_what_every_warp_reads():
    import yskn_b200 as Y
    fn, args_of = Y.lib().yskn_b200_tree_plan, Y.ARGS["tree_plan"]
    for change in (dict(positions="parents"), dict(positions=("starts", 4)), dict(positions=("lens", -16)),
                   dict(mask="parents"), dict(mask="lens"), dict(mask="starts"), dict(mask=("starts", -4)),
                   dict(mask=("starts", 8)), dict(lens=("mask", 36))):
        assert fn(args_of.pack(*apart(TREE_PLAN, **change).values()), None) == Y.EINVAL, change
        assert "arrays of their own" in Y.last_error(), change
    # beside the mask's five rows of two words, and between them where they are far apart
    for change in (dict(lens=("mask", 40)), dict(lens=("mask", -8)), dict(starts=("mask", -12))):
        assert passes(fn, args_of.pack(*apart(TREE_PLAN, **change).values())), change
    far = dict(TREE_PLAN, stride=8)
    for at in range(-16, 5 * 32 + 8, 4):
        args = args_of.pack(*apart(far, lens=("mask", at)).values())
        meets = any(r * 32 < at + 8 and at < r * 32 + 8 for r in range(5))
        assert fn(args, None) == Y.EINVAL if meets else passes(fn, args), at
    one = dict(TREE_PLAN, tokens=1, stride=0)
    assert fn(args_of.pack(*apart(one, lens=("mask", 4)).values()), None) == Y.EINVAL
    assert passes(fn, args_of.pack(*apart(one, lens=("mask", 8)).values()))


def test_tree_accept_refuses_outputs_that_meet_what_every_warp_reads():
    """Results may take the place of the lengths, which a warp reads for its request alone, and what is not wanted may go
    where another result goes."""
    import yskn_b200 as Y
    fn, args_of = Y.lib().yskn_b200_tree_accept, Y.ARGS["tree_accept"]
    for change in [{k: (v, 4)} for k in ("accepted", "lens_out", "next") for v in ("tokens", "parents", "choice", "starts",
                                                                                 "lens")] + [
            dict(path="tokens"), dict(path="parents"), dict(path="choice"), dict(path="starts"), dict(path="lens"),
            dict(path=("starts", -28)), dict(starts=("path", 28))]:
        assert fn(args_of.pack(*apart(TREE_ACCEPT, **change).values()), None) == Y.EINVAL, change
        assert "arrays of their own" in Y.last_error(), change
    for change in (dict(lens_out="lens"), dict(accepted="lens"), dict(next="lens"), dict(accepted="next"),
                   dict(starts=("path", 32)), dict(starts=("path", -12))):
        assert passes(fn, args_of.pack(*apart(TREE_ACCEPT, **change).values())), change
