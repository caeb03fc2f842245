"""CPU: the 8-bit cache's definition, and pages of 8-bit pools shared and copied like bf16 ones."""

import pytest
import torch

from oracle import kv8 as OK
from yapd_amd.paged import PagedKV, SharedPagedKV


def test_codes_are_the_nearest_and_scales_the_largest_value_s():
    x = torch.zeros(6, 64)
    x[0, :4] = torch.tensor([1.0, -1.0, 0.5, 1 / 128])       # 2^0: e = -6, steps of 1/64; half a step goes to the even code
    x[1, :3] = torch.tensor([255.0, 254.0, -255.0])          # e = 1: 127.5 is held to 127
    x[2, :2] = torch.tensor([3.0 / 128, 2.0 ** -130])        # far below the scale
    x[3, :2] = torch.tensor([2.0 ** -130, 2.0 ** -127])      # below the smallest scale's step: codes of 2^-126
    x[4, :3] = torch.tensor([float("inf"), float("nan"), 1.0])
    codes, e = OK.quantise(x)
    assert codes[0, :4].tolist() == [64, -64, 32, 0] and e[0] == 127 - 6
    assert codes[1, :3].tolist() == [127, 127, -127] and e[1] == 127 + 1
    assert codes[2, :2].tolist() == [96, 0] and e[2] == 127 - 12
    assert codes[3, :2].tolist() == [0, 0] and e[3] == 1
    assert codes[4, :3].tolist() == [127, 0, 0] and e[4] == 127 + 121
    assert codes[5].abs().max() == 0 and e[5] == 1


def test_error_is_at_most_half_a_step():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(500, 64, generator=g).bfloat16() * torch.pow(2.0, torch.randint(-60, 60, (500, 1), generator=g))
    codes, e = OK.quantise(x)
    v = OK.values(codes, e)
    half = torch.ldexp(torch.ones(500, dtype=torch.float64), e.int() - 128)
    assert bool(((v - x.double()).abs().amax(-1) <= half).all())
    assert bool((half <= x.double().abs().amax(-1) / 128).all())
    assert torch.equal(v.bfloat16().double(), v)  # every value is a bf16 value


@pytest.mark.parametrize("bits", [8, 16])
def test_pools_by_width(bits):
    kv = PagedKV(n_layers=2, n_rows=2, pages_per_row=3, n_heads=4, device=torch.device("cpu"), kv_bits=bits)
    assert kv.pools[0].shape == (6, 2, 4, 1040 if bits == 8 else 1024)
    assert kv.bytes_per_layer == 6 * 2 * 4 * (1040 if bits == 8 else 2048)


@pytest.mark.parametrize("bits", [0, 4, 32])
def test_other_widths_are_refused(bits):
    for make in (PagedKV, SharedPagedKV):
        with pytest.raises(ValueError, match="kv_bits"):
            make(n_layers=1, n_rows=1, pages_per_row=1, n_heads=4, device=torch.device("cpu"), n_pages=2, kv_bits=bits)


def test_shared_pages_of_an_8_bit_cache():
    """Fork, write to one row's own copy, compact: every row reads what it held."""
    kv = SharedPagedKV(n_layers=2, n_rows=3, pages_per_row=4, n_heads=4, device=torch.device("cpu"), n_pages=12, kv_bits=8)
    g = torch.Generator().manual_seed(1)
    x = torch.randn(40, 4, 64, generator=g).bfloat16()
    codes, scales = OK.quantise(x)

    def write(row, pos):
        for pool in kv.pools:
            for plane in (0, 1):
                OK.write(pool, int(kv.table_host[row, pos // 16]), pos % 16, plane, codes[pos], scales[pos])

    kv.reserve(0, 0, 40)
    for pos in range(40):
        write(0, pos)
    kv.fork(0, [1, 2], 37)
    kv.reserve(1, 20, 21)
    codes[20] = 1
    write(1, 20)
    kv.release(0)
    kv.compact()
    for pool in kv.pools:
        for plane in (0, 1):
            a = OK.read(pool, int(kv.table_host[1, 1]), 4, plane)
            assert torch.equal(a, OK.values(codes[20], scales[20]))
            for pos in (0, 15, 16, 36):
                want = OK.values(codes[pos], scales[pos])
                for row in (1, 2):
                    assert torch.equal(OK.read(pool, int(kv.table_host[row, pos // 16]), pos % 16, plane), want)
