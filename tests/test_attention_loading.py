"""Which warps of the attention's kernel load keys and values: each of them has a box in every stage, so that the ring waits for all that follow it.  Without a device."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def lib():
    from qwengine_b200 import build, load_library
    build.build()
    return load_library()


@pytest.mark.parametrize("pair", [0, 1])
@pytest.mark.parametrize("D", [8, 64, 72, 128, 136, 192, 200, 256])
def test_every_loading_warp_has_a_box(lib, D, pair):
    boxes, warps = C.c_int(), C.c_int()
    for page in (8, 16, 32, 64, 128, 256, 1 << 20):
        rc = lib.q38b_debug_attention_loading(D, page, pair, C.byref(boxes), C.byref(warps))
        if pair and D <= 192:
            assert rc == -1
            continue
        stage = 128 if -(-D // 64) % 2 == 0 else 64                  # elements of a stage
        assert rc == 0 and boxes.value == 128 // min(page, 64 if pair else 128) * (stage // 64)
        assert warps.value == len({box % 3 for box in range(boxes.value)})      # box b is warp b % 3's
        assert boxes.value <= 3 * 32                                           # a lane each


@pytest.mark.gpu
@pytest.mark.parametrize("page", [64, 128, 256])
@pytest.mark.parametrize("D", [64, 128, 192])
def test_one_tile_of_keys_and_many_in_large_pages(ctx, D, page):
    """Stages of one and of two boxes: fewer than warps that load."""
    from test_gpu_cache import run
    for _ in range(3):
        run(ctx, [(1, 1 + 37 * s % 300) for s in range(160)], nq=2, nk=1, D=D, page=page)
        run(ctx, [(1, 5000), (20, 130), (1, 1)], nq=4, nk=1, D=D, page=page)
