"""Refusals of the acceptance of drafted tokens, on the CPU: each argument wrong by itself in a call
that is right but for it."""
import pytest

from ccinfer_amd import _lib

INVALID, UNSUPPORTED = 6, 26
FAKE = 0x10000  # never dereferenced: every call fails validation first


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


# Places of the arguments: inputs, sizes, caches, layers, outputs.
def accept_call(status):
    """(arguments, all pointers different; places) of the entry with or without a status."""
    ins = 7 if status else 6
    names = [f"in{i}" for i in range(ins)] + ["batch", "total", "width", "k", "v", "ks", "vs",
                                              "layers", "stride", "scale_stride", "blocks",
                                              "heads", "dim", "block"] \
        + ["accepted", "nodes", "tokens", "lengths", "stream"]
    at = {n: i for i, n in enumerate(names)}
    args = [FAKE + 4096 * i for i in range(len(names))]
    for n, v in dict(batch=2, total=8, width=4, ks=None, vs=None, layers=2, stride=1 << 20,
                     scale_stride=0, blocks=8, heads=2, dim=64, block=16, stream=None).items():
        args[at[n]] = v
    return args, at


@pytest.mark.parametrize("status", [False, True])
def test_accept_refuses_each_wrong_argument(lib, status):
    f = lib.ccinfer_accept_planned_tokens if status else lib.ccinfer_accept_draft_tokens
    args, at = accept_call(status)

    def code(**change):
        a = list(args)
        for n, v in change.items():
            a[at[n]] = v
        return f(*a)

    # too many requests are refused behind all of these: nothing else is wrong with the call
    assert code(batch=2049) == UNSUPPORTED
    ins = [f"in{i}" for i in range(6)]
    outs = ["accepted", "nodes", "tokens", "lengths"]
    for n in ins + ["k", "v"] + outs:
        assert code(**{n: None}, batch=2049) == INVALID, n
    for n in ("total", "width", "layers", "blocks", "heads", "dim", "block"):
        for v in (0, -1):
            assert code(**{n: v}, batch=2049) == INVALID, (n, v)
    assert code(batch=0) == INVALID and code(batch=-1) == INVALID
    assert code(ks=FAKE, batch=2049) == INVALID and code(vs=FAKE, batch=2049) == INVALID
    assert code(width=1 << 28, batch=2049) == INVALID          # positions past 31 bits
    assert code(stride=8 * 16 * 2 * 64 * 2 - 2, batch=2049) == INVALID
    for out in outs:                                            # an output that is an input
        for n in ins + (["in6"] if status else []):
            assert code(**{out: args[at[n]]}) == INVALID, (out, n)
