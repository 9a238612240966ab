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


def test_tree_plan_refuses_outputs_that_meet_what_every_warp_reads():
    import yskn_b200 as Y
    fn, args_of = Y.lib().yskn_b200_tree_plan, Y.ARGS["tree_plan"]
    for change in (dict(positions="parents"), dict(positions=("starts", 4)), dict(positions=("lens", -16)),
                   dict(mask="parents"), dict(mask="lens"), dict(mask="starts"), dict(mask="positions")):
        assert fn(args_of.pack(*apart(TREE_PLAN, **change).values()), None) == Y.EINVAL, change
        assert "arrays of their own" in Y.last_error(), change


def test_tree_accept_refuses_outputs_that_meet_what_every_warp_reads():
    """The new lengths may take the place of the old ones, which a warp reads for its request alone."""
    import yskn_b200 as Y
    fn, args_of = Y.lib().yskn_b200_tree_accept, Y.ARGS["tree_accept"]
    for change in [{k: (v, 4)} for k in ("accepted", "lens_out", "next") for v in ("tokens", "parents", "choice", "starts",
                                                                                 "lens")] + [
            dict(accepted="lens_out"), dict(next="lens"), dict(next=("accepted", 4)), dict(path="tokens"),
            dict(path="parents"), dict(path="choice"), dict(path="starts"), dict(path="lens")]:
        assert fn(args_of.pack(*apart(TREE_ACCEPT, **change).values()), None) == Y.EINVAL, change
        assert "arrays of their own" in Y.last_error(), change
    # refused for nothing else: the call goes on to the launch, which no machine without a GPU can do
    import torch
    if not torch.cuda.is_available():
        assert fn(args_of.pack(*apart(TREE_ACCEPT, lens_out="lens").values()), None) != Y.EINVAL
