"""Which form a product takes on a device with 148 SMs, so that the GPU tests at
these sizes are known to reach it."""
import pytest

from int8_kernel_lab_b200 import _abi

# (m, n, k, groups), and the form: columns of a tile, pairs, resident b, shares of k
RESIDENT = {(20000, 320, 320, 0): 160, (20011, 333, 330, 0): None, (32768, 100, 450, 0): 128,
            (3001, 2000, 700, 0): 128, (5000, 4096, 384, 0): 256}
PLAIN = [(6000, 1500, 2100, 0), (20000, 1003, 1000, 0), (777, 1111, 1234, 0)]
PAIRS = [(2048, 4096, 4096, 0), (4100, 5000, 4100, 0)]
SPLIT = [(1, 4096, 4096, 0), (3, 70, 16400, 0), (100, 300, 5000, 0)]
GROUPED = [(9000, 1000, 500, 3), (1500, 1408, 1000, 60), (32, 4096, 2048, 32)]


def form(m, n, k, groups, sms=148):
    v = _abi.lib.int8conv_debug_matmul_form(m, n, k, groups, sms)
    return {"columns": v & 0xffff, "pair": bool(v >> 16 & 1), "resident": bool(v >> 17 & 1),
            "shares": v >> 20}


def tiles_per_cta(m, n, k, groups=0, sms=148):
    """Tiles of the busiest CTA (or pair) of a plain launch."""
    f = form(m, n, k, groups)
    columns = -(-n // f["columns"])
    rows = -(-m // (256 if f["pair"] else 128))
    slots = sms // 2 if f["pair"] else sms // columns * columns if f["resident"] else sms
    return -(-rows * columns // slots)


@pytest.mark.parametrize("size", RESIDENT, ids=str)
def test_resident(size):
    f = form(*size)
    assert f["resident"] and not f["pair"] and f["shares"] == 1
    assert RESIDENT[size] in (None, f["columns"])
    assert tiles_per_cta(*size) >= 2


@pytest.mark.parametrize("size", PLAIN, ids=str)
def test_plain(size):
    f = form(*size)
    assert not f["resident"] and not f["pair"] and f["shares"] == 1


@pytest.mark.parametrize("size", PAIRS, ids=str)
def test_pairs(size):
    f = form(*size)
    assert f["pair"] and not f["resident"] and f["shares"] == 1
    assert tiles_per_cta(*size) >= 2


@pytest.mark.parametrize("size", SPLIT, ids=str)
def test_shares_of_k(size):
    assert form(*size)["shares"] in (2, 4, 8)


@pytest.mark.parametrize("size", GROUPED, ids=str)
def test_grouped(size):
    f = form(*size)
    assert not f["resident"] and f["shares"] == 1


@pytest.mark.parametrize("size", [(0, 1, 1, 0), (1, 0, 1, 0), (1, 1, 0, 0), (1, 1, 131072, 0),
                                  (1 << 31, 1, 1, 0), (1, 1, 1, 1025), (1, 1, 1, -1)], ids=str)
def test_sizes_out_of_range(size):
    assert _abi.lib.int8conv_debug_matmul_form(*size, 148) == 0
    assert _abi.lib.int8conv_debug_matmul_form(1, 1, 1, 0, 0) == 0
