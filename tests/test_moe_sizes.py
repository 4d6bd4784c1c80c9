"""Sizes at the ends of the argument types of the mixture-of-experts entry points: refused or answered, before anything reaches a GPU."""
import ctypes

import pytest

import awesome_fusion_b200 as pkg

E_LARGE = -6
PTR = 0x10000


@pytest.fixture(scope="module")
def lib():
    return pkg.load()


@pytest.mark.parametrize("tokens", [(1 << 31) - 1, 1 << 31, (1 << 32) - 256, (1 << 32) - 255, (1 << 32) - 1])
def test_route_workspace_of_huge_batches(lib, tokens):
    """The size is a division by the tokens of a block; rounded up in 32 bits those would be 0 from 2^32 - 255 tokens on."""
    n = ctypes.c_uint64(7)
    rc = lib.lib.afb_moe_route_workspace(tokens, 64, ctypes.byref(n))
    if tokens >> 31:
        assert rc == E_LARGE and n.value == 7
    else:
        assert rc == 0 and 0 < n.value <= 256 * 64 * 4


@pytest.mark.parametrize("changes", [dict(tokens=1 << 31), dict(tokens=(1 << 32) - 65535), dict(tokens=(1 << 32) - 1), dict(n=1 << 31, ld_out=1 << 31, ld_y=1 << 31)])
def test_combine_of_huge_batches(lib, changes):
    """A block walks tokens in strides of up to 65535: with more than 2^32 - 65535 of them the walk would pass 32 bits and begin again, for ever."""
    args = lib.make_moe_combine_args(PTR, 2 * PTR, PTR, PTR, tokens=10, top_k=1, rows=20, n=8)
    for name, value in changes.items():
        setattr(args, name, value)
    assert lib.moe_combine_launch_status(args) == E_LARGE
