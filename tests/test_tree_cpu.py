"""CPU: masks of drafted trees, and what attn_tree, kv8_write, kv8_unpack and kv_keep refuse (before any GPU call)."""

import ctypes

import numpy as np
import pytest
import torch

from oracle import tree as OT
from yapd_amd import kernels

P = 4096  # stands for a 16-byte aligned device address, never read: refused calls launch nothing
EINVAL = 1


def test_tree_masks_name_a_node_and_its_ancestors():
    m = kernels.tree_masks([-1, 0, 0, 2, -1, 4, 3])
    assert m.dtype == np.int64 and m.tolist() == [0b1, 0b11, 0b101, 0b1101, 0b10000, 0b110000, 0b1001101]
    assert kernels.tree_masks([]).shape == (0,)
    chain = kernels.tree_masks(range(-1, 63)).view(np.uint64)
    assert int(chain[63]) == 2**64 - 1


@pytest.mark.parametrize("parents", [[0], [-1, 1], [-1, -2], [-1] * 65])
def test_tree_masks_refuses(parents):
    with pytest.raises(ValueError):
        kernels.tree_masks(parents)


def test_oracle_chain_is_causal():
    see = OT.visible(9, 4, [1, 3, 7, 15], None, 0)
    assert torch.equal(see, torch.arange(9)[None] <= torch.arange(5, 9)[:, None])
    windowed = OT.visible(9, 4, [1, 3, 7, 15], 4, 1)
    pos = torch.arange(5, 9)[:, None]
    j = torch.arange(9)[None]
    assert torch.equal(windowed, (j <= pos) & ((j < 1) | (j > pos - 4)))


def tree(**over):
    a = dict(q=P, tok=1024, pool=P, bits=8, pages=100, table=P, stride=8, cols=8, kv_len=P, q_start=None, mask=P, rows=2,
             max_q=3, n_q=6, heads=16, window=64, sinks=0, max_kv=100, scale=0.125, ws=None, floats=0, out=1 << 40, stream=None)
    a.update(over)
    return list(a.values())


@pytest.mark.parametrize("over,msg", [
    (dict(q=None), b"NULL"), (dict(mask=None), b"NULL"), (dict(out=None), b"NULL"), (dict(kv_len=None), b"NULL"),
    (dict(bits=4), b"bits"), (dict(max_q=65, n_q=130, window=100), b"64 nodes"), (dict(max_q=0), b"max_q"),
    (dict(rows=0), b"rows"), (dict(heads=6), b"multiple of 4"), (dict(heads=0), b"multiple of 4"),
    (dict(window=2), b"window"), (dict(sinks=-1), b"sinks"), (dict(max_kv=0), b"max_kv"), (dict(q=P + 2), b"aligned"),
    (dict(out=P + 8), b"aligned"), (dict(tok=1020), b"q_tok_stride"), (dict(tok=960), b"q_tok_stride"),
    (dict(cols=0), b"empty"), (dict(stride=7), b"empty"), (dict(pages=0), b"empty"), (dict(n_q=7), b"rows * max_q"),
    (dict(scale=0.0), b"scale"), (dict(scale=float("nan")), b"scale"), (dict(scale=-1.0), b"scale"),
    (dict(out=P), b"overlaps"), (dict(q=1 << 41, out=P + 2 * 1040 * 16 * 99), b"overlaps the pool"),
    (dict(rows=1 << 20, n_q=3 << 20), b"too many rows"),
    (dict(rows=1, n_q=3, max_kv=10000, cols=700, stride=700, window=2**30), b"workspace"),
])
def test_attn_tree_refuses(over, msg):
    lib = kernels.load_library()
    assert lib.yapd_attn_tree(*tree(**over)) == EINVAL
    assert msg in lib.yapd_last_error()


def test_attn_tree_workspace():
    need = kernels.load_library().yapd_attn_tree_workspace
    assert need(256, 1, 256, 16, 2**30, 0, 4000, 8) == 0
    assert need(1, 3, 3, 16, 2**30, 0, 30000, 16) % (3 * 16 * 66) == 0 < need(1, 3, 3, 16, 2**30, 0, 30000, 16)
    assert need(1, 65, 65, 16, 2**30, 0, 30000, 16) == -1
    assert need(1, 3, 3, 16, 2, 0, 30000, 16) == -1


WRITE = dict(k=P, v=P, ks=1024, vs=1024, pool=P, pages=9, table=P, stride=4, cols=4, pos0=P, q_start=None, rows=3, n=6,
             heads=16, stream=None)


@pytest.mark.parametrize("over,msg", [
    (dict(k=None), b"NULL"), (dict(pos0=None), b"NULL"), (dict(v=P + 8), b"aligned"), (dict(rows=0), b"empty"),
    (dict(n=0), b"empty"), (dict(pages=0), b"empty"), (dict(heads=5), b"multiple of 4"), (dict(ks=1020), b"strides"),
    (dict(vs=512), b"strides"), (dict(cols=0), b"table"), (dict(stride=3), b"table"), (dict(n=7), b"multiple of rows"),
    (dict(rows=1, n=2**31 - 1, heads=1024, ks=65536, vs=65536), b"too many"),
])
def test_kv8_write_refuses(over, msg):
    lib = kernels.load_library()
    assert lib.yapd_kv8_write(*dict(WRITE, **over).values()) == EINVAL
    assert msg in lib.yapd_last_error()


UNPACK = dict(pool8=P, pages8=9, table8=P, stride8=4, cols8=4, kv_len=P, rows=3, max_kv=64, heads=16, pool=1 << 40, pages=9,
              table=P, stride=4, cols=4, stream=None)


@pytest.mark.parametrize("over,msg", [
    (dict(pool8=None), b"NULL"), (dict(kv_len=None), b"NULL"), (dict(pool=P + 8), b"aligned"), (dict(rows=0), b"rows"),
    (dict(rows=65536), b"rows"), (dict(max_kv=0), b"max_kv"), (dict(heads=6), b"multiple of 4"), (dict(cols8=0), b"table"),
    (dict(stride=3), b"table"), (dict(pool=P), b"overlap"), (dict(pool=P + 1040 * 32 * 9 - 16), b"overlap"),
    (dict(pool8=P + 2048 * 32 * 9 - 16, pool=P), b"overlap"),
    (dict(rows=65535, max_kv=2**20, cols=65535, stride=65535, cols8=65535, stride8=65535), b"too many"),
])
def test_kv8_unpack_refuses(over, msg):
    lib = kernels.load_library()
    assert lib.yapd_kv8_unpack(*dict(UNPACK, **over).values()) == EINVAL
    assert msg in lib.yapd_last_error()


@pytest.mark.parametrize("over,msg", [
    (dict(table=None), b"NULL"), (dict(n_kept=None), b"NULL"), (dict(bits=32), b"bits"), (dict(layers=0), b"layers"),
    (dict(rows=0), b"rows"), (dict(rows=65536), b"rows"), (dict(heads=7), b"multiple of 4"), (dict(max_kept=65, kept_stride=65), b"64"),
    (dict(max_kept=0), b"64"), (dict(kept_stride=3), b"64"), (dict(cols=0), b"table"), (dict(stride=2), b"table"),
])
def test_kv_keep_refuses(over, msg):
    pools = (ctypes.c_void_p * 2)(P, P + 16)
    a = dict(pools=pools, layers=2, bits=8, pages=9, heads=16, table=P, stride=4, cols=4, base=P, kept=P, kept_stride=4,
             max_kept=4, n_kept=P, rows=3, stream=None)
    a.update(over)
    lib = kernels.load_library()
    assert lib.yapd_kv_keep(*a.values()) == EINVAL
    assert msg in lib.yapd_last_error()
    pools[1] = P + 8
    assert lib.yapd_kv_keep(*dict(a, table=P, n_kept=P, bits=8, layers=2, rows=3, heads=16, max_kept=4, kept_stride=4, cols=4,
                                  stride=4).values()) == EINVAL
    assert b"layer 1" in lib.yapd_last_error()


@pytest.mark.parametrize("bits,tile", [(8, 1040), (16, 2048)])
def test_kv_keep_refuses_a_pool_given_twice(bits, tile):
    size = 9 * 2 * 16 * tile
    lib = kernels.load_library()
    for addresses in ((P, P), (P, P + size, P + size - 16), (P + size - 16, P + 2 * size, P)):
        pools = (ctypes.c_void_p * len(addresses))(*addresses)
        assert lib.yapd_kv_keep(pools, len(addresses), bits, 9, 16, P, 4, 4, P, P, 4, 4, P, 3, None) == EINVAL
        assert b"overlap" in lib.yapd_last_error()


def test_kv8_copy_pages_refuses():
    pools = (ctypes.c_void_p * 1)(P)
    ids = (ctypes.c_int32 * 2)(1, 9)
    lib = kernels.load_library()
    assert lib.yapd_kv8_copy_pages(pools, 1, 9, 16, ids, ids, 2, None) == EINVAL
    assert b"kv8_copy_pages: pair 1" in lib.yapd_last_error()


def test_wrappers_refuse_cpu_tensors():
    x = torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    t = torch.zeros(2, 4, dtype=torch.int32)
    p8 = torch.zeros(8, 2, 4, 1040, dtype=torch.uint8)
    with pytest.raises(ValueError, match="GPU"):
        kernels.attn_tree(x, p8, t, i, torch.zeros(2, 3, dtype=torch.int64), x.clone(), 0.125)
    with pytest.raises(ValueError, match="GPU"):
        kernels.kv8_write(x[0], x[0], p8, t, i)
    with pytest.raises(ValueError, match="GPU"):
        kernels.kv8_unpack(p8, t, i, torch.zeros(8, 2, 4, 1024, dtype=torch.bfloat16), t)
    with pytest.raises(ValueError, match="GPU"):
        kernels.kv_keep([p8], t, i, t, i)
