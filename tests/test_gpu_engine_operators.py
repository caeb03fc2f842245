"""GPU: windowed attention, page copies and token log probabilities on what the engine makes: its cache, its rotated queries and
its captured logits."""

import pytest
import torch

from oracle import logprob as OL
from oracle import window as OW
from tests._window_cases import tolerance
from yapd_amd import kernels, scoring
from yapd_amd.engines.hip import HipEngine
from yapd_amd.synthetic import make_t3

pytestmark = pytest.mark.gpu
LENS, BL, SCALE = [90, 200, 333], 16, 0.125


@pytest.fixture(scope="module")
def world(dev):
    model = make_t3(n_layers=2, seed=21, norm_jitter=True, device=dev)
    eng = HipEngine(model, 512, torch.bfloat16, batch_size=3, page_table_seed=3)
    g = torch.Generator().manual_seed(5)
    sos = eng.prefix_forward([torch.randn(1, n, 1024, generator=g).bfloat16().to(dev) for n in LENS])
    block = torch.randn(3, BL, 1024, generator=g).bfloat16().to(dev)
    return model, eng, sos, block


@pytest.mark.parametrize("window,sinks", [(10000, 0), (64, 0), (100, 20), (17, 4)])
def test_windowed_attention_on_the_engines_cache(world, dev, window, sinks):
    _, eng, _, block = world
    layer = eng.layer_forward(0, block, LENS)  # writes the block's K and V behind the prefixes
    kv = [n + BL for n in LENS]
    out = torch.empty_like(layer["q"])
    kernels.attn_window(layer["q"], eng.kv.pools[0], eng.kv.table, torch.tensor(kv, dtype=torch.int32, device=dev), out, SCALE,
                        window=window, sinks=sinks, causal=False)
    for r, n in enumerate(kv):
        K, V = kernels.kv_gather(eng.kv.pools[0], eng.kv.table[r].contiguous(), n)
        want, a = OW.attend(layer["q"][r].cpu(), K.cpu(), V.cpu(), window, sinks, False, SCALE)
        assert bool(((out[r].cpu().double() - want).abs() <= tolerance(want, a)).all()), r
        if window > n:  # the engine's own attention, held to the same bound
            own = layer["attn"][r].view(BL, 16, 64).cpu().double()
            assert bool(((own - want).abs() <= tolerance(want, a)).all()), r


def test_a_row_whose_pages_were_copied_decodes_alike(world):
    """Row 0 as a copy of row 2's prefix: the same block gives the same hidden states, bit for bit."""
    _, eng, _, block = world
    same = block[2:].expand(3, -1, -1).contiguous()
    was = [p.clone() for p in eng.kv.pools]
    eng.kv.copy_row_pages(2, 0, LENS[2])
    hidden = eng.block_forward(same, [LENS[2], LENS[1], LENS[2]])
    assert torch.equal(hidden[0], hidden[2]) and not torch.equal(hidden[1], hidden[2])
    for p, w in zip(eng.kv.pools, was):
        p.copy_(w)


def test_token_logprobs_of_captured_logits(world, dev):
    """The padded logits of the captured step as they are, replayed on two blocks."""
    model, eng, sos, block = world
    eng.capture_cuda_graph(BL, speech_head=model.speech_head)
    eng.set_shift_ctx(sos.view(3, 1, -1))
    tokens = torch.randint(-1, 8194, (3, BL), generator=torch.Generator().manual_seed(2))
    for emb in (block, block.flip(0)):
        _, logits = eng.block_forward_graph(emb, LENS)
        assert logits.shape == (3, BL, 8194) and logits.stride(1) == 8200
        res = scoring.token_logprobs(logits, tokens.to(dev), top_k=8)
        x = logits.reshape(-1, 8194).cpu()
        lp, ent, top_lp, top = OL.token_logprobs(x, tokens.view(-1), 8)
        tol, tol_e = OL.tolerances(x, ent)
        u = 2.0 ** -24
        assert bool(((res.logprob.cpu().double().view(-1) - lp).abs() <= tol + u * lp.abs()).all())
        assert bool(((res.entropy.cpu().double().view(-1) - ent).abs() <= tol_e + u * ent).all())
        assert torch.equal(res.top_token.cpu().view(-1, 8), top)
        assert bool(((res.top_logprob.cpu().double().view(-1, 8) - top_lp).abs() <= tol[:, None] + u * top_lp.abs()).all())
