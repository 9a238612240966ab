"""Outputs of the call that forks requests that would meet what other CTAs still read: refused with EINVAL and a message before any device work (fake, never dereferenced pointers; no GPU)."""
from test_tree_abi import BATCH_EDIT, P


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
