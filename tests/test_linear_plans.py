"""Plans of dense products: the launches that they make are ones that can be made."""
import ctypes
import os
import sys

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "awesome-cute_amd"))
import streamk  # noqa: E402

MOST = 2 ** 32 - 1  # threads of a launch


def threads(plan, m, n, gated):
    rows, cols, slices = plan
    if m <= 64 and cols <= 32:
        return -(-n // (cols // (2 if gated == 1 else 1))) * 256
    columns = -(-n // 16) * 32 if gated == 1 else n
    return -(-m // rows) * -(-columns // cols) * slices * (256 if cols <= 64 or rows >= 160 else 512)


def test_launches_of_the_plans():
    rng, most = np.random.default_rng(0), 0
    for at in range(6000):
        m, n = int(2 ** rng.uniform(0, 30.9)), 8 * max(1, int(2 ** rng.uniform(0, 18)))
        k = 8 * max(1, int(2 ** rng.uniform(0, 10)))
        gated, turned = ((0, 0), (1, 0), (2, 0), (0, 1), (0, 2))[at % 5]
        if turned == 2:
            m = 8 * max(1, m // 8)
        if gated == 1:
            n = min(n, 1 << 17)
        try:
            plan = streamk.product_plan(m, n, k, gated, turned)
        except ValueError as error:
            assert "too many" in str(error)
            # not even by tiles of 256 x 256
            assert threads((256, 256, 1), m, n, gated) > MOST
            continue
        count = threads(plan, m, n, gated)
        most = max(most, count)
        assert count <= MOST, (m, n, k, gated, turned, plan)
    assert most > 2 ** 30


def test_launches_at_the_limit():
    # tiles of 64 x 64 would be 2^24 workgroups of 256 threads, one thread too many
    assert threads(streamk.product_plan(1 << 30, 8, 8), 1 << 30, 8, 0) <= MOST
    assert threads(streamk.product_plan((1 << 30) - 64, 8, 8), (1 << 30) - 64, 8, 0) <= MOST
    for gated in (0, 2):
        with pytest.raises(ValueError, match="too many"):
            streamk.product_plan(0x7ffffe00, 1024, 64, gated)
        with pytest.raises(ValueError, match="too many"):
            streamk.product_plan(0x7fffffff, 8, 64, gated)
    try:
        streamk.force_product_tile(64, 64)
        with pytest.raises(ValueError, match="too many"):
            streamk.product_plan(1 << 30, 8, 8)
        assert streamk.product_plan(1 << 29, 8, 8)[:2] == (64, 64)
    finally:
        streamk.force_product_tile(0)


def test_refusals_of_the_entries():
    """Host checks alone: no GPU is asked for anything."""
    lib, L, P = streamk._lib, ctypes.c_longlong, ctypes.c_void_p
    for m, n in ((0x7fffffff, 8), (0x7ffffe00, 1024), (1 << 28, 1 << 16)):
        assert lib.feedforward_product(P(16), P(16), P(16), m, n, 8, L(8), L(8), L(n), 0, 0, None, L(0), 0, None) == 1
        assert b"too many" in lib.feedforward_last_error()
        assert lib.feedforward_linear(P(16), P(16), P(16), None, None, None, m, n, 8, L(8), L(8), L(n), L(0), L(0), 0, 1, None,
                                      None, L(0), 0, None) == 1
        assert b"too many" in lib.feedforward_last_error()
        assert lib.feedforward_gated(P(16), P(16), P(16), None, m, n, 8, L(8), L(8), L(n), L(0), 0, 1, None, L(0), 0, None) == 1
        assert b"too many" in lib.feedforward_last_error()
    # rows of eight columns a thread
    assert lib.feedforward_gated_grad(P(16), P(16), P(16), 1 << 28, 128, L(128), L(256), L(256), 0, 1, 0, None) == 1
    assert b"too many" in lib.feedforward_last_error()


def test_the_kernel_for_few_rows_and_the_small_tiles_of_its_name():
    """A tile of 32 x 32 of more than 64 rows is no other kernel's."""
    try:
        streamk.force_product_tile(32, 32)
        assert streamk.product_plan(64, 520, 192, 2) == (64, 32, 1) and streamk.product_plan(65, 520, 192, 2)[:2] == (32, 32)
        assert streamk.product_plan(65, 520, 192)[:2] != (32, 32)
        streamk.force_product_tile(16, 16)
        assert streamk.product_plan(64, 520, 192, 2) == (64, 16, 1) and streamk.product_plan(65, 520, 192, 2)[1] >= 32
    finally:
        streamk.force_product_tile(0)
