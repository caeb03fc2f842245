"""Loader and typed wrappers for the native gfx950 library ``libyapd_t3.so``.

The counterpart of the reference's native-kernel convention in
server/kernels.py:103-165: the library is loaded once (``lru_cache``, as
``load_snake_extension`` at server/kernels.py:103-106), every wrapper checks
its tensors before launching (as the ``TORCH_CHECK``s of
server/kernels.py:69-75), launches on the caller's current stream
(server/kernels.py:79) and lets the caller own the outputs.  Unlike
server/kernels.py:110-112 there is no torch fallback: a missing library or
a failed precondition raises.
"""

from __future__ import annotations

import ctypes
import functools
from array import array
from pathlib import Path
from typing import Optional

import torch

LIB_PATH = Path(__file__).resolve().parent / "_lib" / "libyapd_t3.so"

c_int, c_i64, c_u64, c_float, c_size, c_void = (
    ctypes.c_int, ctypes.c_int64, ctypes.c_uint64, ctypes.c_float, ctypes.c_size_t, ctypes.c_void_p)

# name -> (restype, argtypes); mirrors include/yapd_t3.h, yapd_probe.h and yapd_vocoder.h.
_SIGNATURES = {
    "yapd_last_error": (ctypes.c_char_p, []),
    "yapd_abi_version": (c_int, []),
    "yapd_score_cfg_pmi_unmask": (c_int, [
        c_void, c_i64, c_i64, c_int, c_int, c_int, c_int, c_int, c_int, c_int,
        c_void, c_void, c_void, c_void, c_void, c_void, c_int, c_float, c_int, c_i64, c_i64,
        c_float, c_int, c_u64, c_u64, c_void, c_void, c_void, c_void, c_void, c_void, c_void]),
    "yapd_token_logprobs": (c_int, [c_void, c_int, c_i64, c_i64, c_int, c_int, c_int, c_void, c_int, c_void, c_void,
                                    c_void, c_void, c_void]),
    "yapd_sample_tokens": (c_int, [c_void, c_int, c_i64, c_i64, c_int, c_int, c_int, c_void, c_void, c_float, c_void,
                                   c_int, c_void, c_float, c_void, c_float, c_void, c_void, c_void]),
    "yapd_attn_plan": (c_int, [c_void, c_int, c_int, c_int, c_void, c_int, c_void, c_int, c_void, c_void, c_void]),
    "yapd_attn_paged_block": (c_int, [
        c_void, c_void, c_i64, c_void, c_int, c_int, c_void, c_int, c_int, c_int, c_void, c_int, c_void, c_int,
        c_void, c_void, c_void, c_int, c_float, c_int, c_void, c_void]),
    "yapd_attn_paged_block_noalloc": (c_int, [
        c_void, c_void, c_i64, c_void, c_int, c_int, c_void, c_int, c_int, c_int, c_void, c_int, c_void, c_int,
        c_void, c_int, c_float, c_int, c_void, c_void]),
    "yapd_attn_window": (c_int, [
        c_void, c_i64, c_void, c_i64, c_void, c_int, c_int, c_void, c_void, c_int, c_int, c_int, c_int, c_int, c_int,
        c_int, c_int, c_float, c_void, c_i64, c_void, c_void]),
    "yapd_attn_window_workspace": (c_i64, [c_int, c_int, c_int, c_int, c_int, c_int, c_int, c_int]),
    "yapd_kv_write": (c_int, [c_void, c_void, c_i64, c_i64, c_void, c_i64, c_void, c_int, c_int, c_void, c_int,
                              c_int, c_int, c_void]),
    "yapd_kv_gather": (c_int, [c_void, c_i64, c_void, c_int, c_int, c_int, c_void, c_void, c_void]),
    "yapd_kv_copy_pages": (c_int, [c_void, c_int, c_i64, c_int, c_void, c_void, c_int, c_void]),
    "yapd_kv8_copy_pages": (c_int, [c_void, c_int, c_i64, c_int, c_void, c_void, c_int, c_void]),
    "yapd_kv8_write": (c_int, [c_void, c_void, c_i64, c_i64, c_void, c_i64, c_void, c_int, c_int, c_void, c_void, c_int,
                               c_int, c_int, c_void]),
    "yapd_kv8_unpack": (c_int, [c_void, c_i64, c_void, c_int, c_int, c_void, c_int, c_int, c_int, c_void, c_i64, c_void,
                                c_int, c_int, c_void]),
    "yapd_kv_keep": (c_int, [c_void, c_int, c_int, c_i64, c_int, c_void, c_int, c_int, c_void, c_void, c_int, c_int,
                             c_void, c_int, c_void]),
    "yapd_attn_tree": (c_int, [
        c_void, c_i64, c_void, c_int, c_i64, c_void, c_int, c_int, c_void, c_void, c_void, c_int, c_int, c_int, c_int,
        c_int, c_int, c_int, c_float, c_void, c_i64, c_void, c_void]),
    "yapd_attn_tree_workspace": (c_i64, [c_int, c_int, c_int, c_int, c_int, c_int, c_int, c_int]),
    "yapd_gemm_bf16": (c_int, [c_void, c_i64, c_void, c_i64, c_int, c_int, c_int, c_void, c_i64, c_void]),
    "yapd_gemm_bf16_residual": (c_int, [c_void, c_i64, c_void, c_i64, c_int, c_int, c_int, c_void, c_i64, c_void]),
    "yapd_gemm_head_shift": (c_int, [c_void, c_void, c_int, c_int, c_int, c_void, c_i64, c_int, c_void, c_i64,
                                     c_void]),
    "yapd_gemm_swiglu": (c_int, [c_void, c_i64, c_void, c_int, c_int, c_int, c_void, c_i64, c_void]),
    "yapd_gemm_qkv_rope_kv": (c_int, [c_void, c_i64, c_void, c_int, c_int, c_int, c_void, c_void, c_int, c_void,
                                      c_int, c_void, c_void, c_i64, c_void, c_int, c_int, c_void]),
    "yapd_rmsnorm": (c_int, [c_void, c_void, c_void, c_void, c_float, c_int, c_int, c_void, c_void]),
    "yapd_gemm_rmsnorm_qkv_rope_kv": (c_int, [c_void, c_void, c_float, c_void, c_void, c_int, c_int, c_int, c_void,
                                              c_void, c_int, c_void, c_int, c_void, c_void, c_i64, c_void, c_int,
                                              c_int, c_void]),
    "yapd_qgemm_affine": (c_int, [c_void, c_i64, c_void, c_void, c_void, c_int, c_int, c_int, c_int, c_int,
                                  c_void, c_i64, c_void]),
    "yapd_dequant_affine": (c_int, [c_void, c_void, c_void, c_int, c_int, c_int, c_int, c_void, c_void]),
    "yapd_mfma_peak_probe": (c_int, [c_int, c_int, c_int, c_void, c_void]),
    "yapd_hbm_read_probe": (c_int, [c_void, c_i64, c_int, c_void, c_void]),
    "yapd_tick_update": (c_int, [c_int, c_int, c_int, c_int, c_int, c_i64, c_i64, c_i64, c_i64, c_void, c_i64,
                                 c_void, c_void, c_void, c_void, c_void, c_void, c_void, c_void, c_void, c_void,
                                 c_void, c_void]),
    "yapd_t3_block_forward": (c_int, [c_void, c_void, c_void, c_int, c_int, c_void, c_void, c_int, c_void,
                                      c_void, c_int, c_void, c_void, c_i64, c_void]),
    "yapd_t3_prefill_packed": (c_int, [c_void, c_void, c_void, c_int, c_int, c_int, c_void, c_void, c_void, c_void,
                                       c_void, c_void]),
    # include/yapd_vocoder.h
    "yapd_snake": (c_int, [c_void, c_void, c_void, c_void, c_i64, c_int, c_i64, c_void]),
    "yapd_residual_bias": (c_int, [c_void, c_void, c_void, c_void, c_i64, c_int, c_i64, c_void]),
    "yapd_mean3": (c_int, [c_void, c_void, c_void, c_void, c_i64, c_void]),
    "yapd_residual_bias_snake": (c_int, [c_void, c_void, c_void, c_void, c_void, c_void, c_i64, c_int, c_i64,
                                         c_void]),
    "yapd_branch_start": (c_int, [c_void, c_void, c_void, c_void, c_void, c_void, c_void, c_void, c_void, c_i64,
                                  c_int, c_i64, c_void]),
    "yapd_voc_stitch": (c_int, [c_void, c_i64, c_i64, c_int, c_void, c_int, c_void, c_void, c_int, c_void, c_int,
                                c_void, c_int, c_void, c_int, c_void, c_i64, c_void]),
}

STITCH_JOB_INTS = 12  # YAPD_STITCH_JOB_INTS of include/yapd_vocoder.h


class T3QWeight(ctypes.Structure):
    """``yapd_t3_qweight`` of include/yapd_t3.h (MLX-layout codes, fp16 scales and biases)."""
    _fields_ = [("packed", c_void), ("scales", c_void), ("biases", c_void)]


class T3Layer(ctypes.Structure):
    """``yapd_t3_layer`` of include/yapd_t3.h (``qbits`` 0: the bf16 weights; 4 or 8: ``q_*``)."""
    _fields_ = [("w_qkv", c_void), ("w_o", c_void), ("w_gate_up", c_void), ("w_down", c_void),
                ("ln_in", c_void), ("ln_post", c_void), ("eps_in", c_float), ("eps_post", c_float),
                ("kv_pool", c_void), ("qbits", c_int), ("q_qkv", T3QWeight), ("q_o", T3QWeight),
                ("q_gate_up", T3QWeight), ("q_down", T3QWeight)]


class T3Model(ctypes.Structure):
    """``yapd_t3_model`` of include/yapd_t3.h."""
    _fields_ = [("n_layers", c_int), ("hidden", c_int), ("n_heads", c_int), ("ffn", c_int),
                ("layers", ctypes.POINTER(T3Layer)), ("final_norm", c_void), ("final_eps", c_float),
                ("rope_cos", c_void), ("rope_sin", c_void), ("rope_positions", c_int), ("n_pages", c_i64),
                ("page_table", c_void), ("table_stride", c_int), ("table_cols", c_int)]


class T3Workspace(ctypes.Structure):
    """``yapd_t3_workspace`` of include/yapd_t3.h."""
    _fields_ = [("residual", c_void), ("q", c_void), ("attn", c_void), ("normed", c_void), ("delta", c_void),
                ("act", c_void), ("work", c_void), ("n_work", c_int), ("merge", c_void), ("n_merge", c_int),
                ("counts", c_void), ("part_o", c_void), ("part_ml", c_void), ("n_slots", c_int),
                ("wdq", c_void), ("wdq_elems", c_i64)]


class HipKernelError(RuntimeError):
    """A native entry point returned a nonzero status."""


def library_built() -> bool:
    return LIB_PATH.exists()


@functools.lru_cache(maxsize=1)
def load_library() -> ctypes.CDLL:
    """Load ``libyapd_t3.so`` once; raise ``ImportError`` if it was never built."""
    if not LIB_PATH.exists():
        raise ImportError(f"{LIB_PATH} is missing; build it with `python -m yapd_amd.build`")
    lib = ctypes.CDLL(str(LIB_PATH))
    for name, (res, args) in _SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    return lib


def check(rc: int) -> None:
    if rc != 0:
        msg = load_library().yapd_last_error().decode(errors="replace")
        if rc == 1:
            raise ValueError(msg)
        raise HipKernelError(msg)


def stream_ptr(device: torch.device) -> int:
    # the raw handle: building a torch.cuda.Stream object costs more than the launch it is for
    if device.index is not None:
        return torch._C._cuda_getCurrentRawStream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


def ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def require(cond: bool, msg: str) -> None:
    if not cond:
        raise ValueError(msg)


def require_cuda(t: torch.Tensor, name: str, dtype: torch.dtype, device: torch.device,
                 contiguous: bool = True) -> None:
    # one test on the way of every call; the messages are formatted only for a tensor that fails it
    if t.is_cuda and t.dtype == dtype and t.device == device and (not contiguous or t.is_contiguous()):
        return
    require(t.is_cuda, f"{name} must be a GPU tensor")
    require(t.device == device, f"{name} is on {t.device}, expected {device}")
    require(t.dtype == dtype, f"{name} must be {dtype}, got {t.dtype}")
    require(t.is_contiguous(), f"{name} must be contiguous")


# --------------------------------------------------------------------------- #
# (c) scoring
# --------------------------------------------------------------------------- #

def score_cfg_pmi_unmask(
    logits: torch.Tensor, *, n_pairs: int, cond_row0: int, pair_row_step: int,
    null_row_offset: Optional[int], log_prior: torch.Tensor, xt_blk: torch.Tensor,
    k_step: torch.Tensor, sched: torch.Tensor, q_tab: torch.Tensor, cfg_w: float,
    quantile_on: bool, mask_id: int, stop_id: int, out: dict, active: Optional[torch.Tensor] = None, temperature: float = 0.0,
    pos_gumbel: bool = False, seed: int = 0, rng_offset: int = 0,
) -> None:
    """Launch the scoring kernel; results land in the tensors of ``out``.

    ``logits`` is bf16 ``[rows, bl, V]`` with a unit last stride (a padded
    row pitch is fine); ``out`` holds ``sampled`` (int64), ``pmi`` (fp32),
    ``unmask`` (uint8), ``xt_out`` (int64) of shape ``[n_pairs, bl]`` and
    ``n_mask_after`` (int32), ``hit_eos`` (uint8) of shape ``[n_pairs]``.
    """
    lib = load_library()
    dev = logits.device
    require_cuda(logits, "logits", torch.bfloat16, dev, contiguous=False)
    require(logits.dim() == 3 and logits.stride(2) == 1, "logits must be [rows, bl, V] with unit last stride")
    rows, bl, V = logits.shape
    last_row = cond_row0 + (n_pairs - 1) * pair_row_step + max(0, null_row_offset or 0)
    if not (0 <= cond_row0 and last_row < rows):
        raise ValueError(f"pair layout reaches row {last_row} of {rows}")
    require(null_row_offset is None or cond_row0 + null_row_offset >= 0, "null rows out of range")
    require_cuda(log_prior, "log_prior", torch.float32, dev)
    require(log_prior.numel() == V, "log_prior must have V entries")
    require_cuda(xt_blk, "xt_blk", torch.int64, dev)
    if not (tuple(xt_blk.shape) == (n_pairs, bl)):
        raise ValueError(f"xt_blk must be [{n_pairs}, {bl}]")
    require_cuda(k_step, "k_step", torch.int64, dev)
    require(k_step.numel() == n_pairs, "k_step must have n_pairs entries")
    require_cuda(sched, "sched", torch.int32, dev)
    require_cuda(q_tab, "q_tab", torch.float32, dev)
    require(sched.numel() == q_tab.numel() and sched.numel() >= 1, "sched/q_tab must both have K entries")
    if active is not None:
        require_cuda(active, "active", torch.uint8, dev)
        require(active.numel() == n_pairs, "active must have n_pairs entries")
    for name, dt, shape in (("sampled", torch.int64, (n_pairs, bl)), ("pmi", torch.float32, (n_pairs, bl)),
                            ("unmask", torch.uint8, (n_pairs, bl)), ("xt_out", torch.int64, (n_pairs, bl)),
                            ("n_mask_after", torch.int32, (n_pairs,)), ("hit_eos", torch.uint8, (n_pairs,))):
        t = out[name]
        require_cuda(t, name, dt, dev)
        if not (tuple(t.shape) == shape):
            raise ValueError(f"{name} must be {shape}")
    check(lib.yapd_score_cfg_pmi_unmask(
        logits.data_ptr(), logits.stride(0), logits.stride(1), n_pairs, bl, V,
        cond_row0, pair_row_step, 0 if null_row_offset is None else 1, null_row_offset or 0,
        log_prior.data_ptr(), xt_blk.data_ptr(), k_step.data_ptr(), ptr(active),
        sched.data_ptr(), q_tab.data_ptr(), sched.numel(), float(cfg_w), int(bool(quantile_on)),
        int(mask_id), int(stop_id), float(temperature), int(bool(pos_gumbel)),
        int(seed) & (2**64 - 1), int(rng_offset) & (2**64 - 1),
        out["sampled"].data_ptr(), out["pmi"].data_ptr(), out["unmask"].data_ptr(),
        out["xt_out"].data_ptr(), out["n_mask_after"].data_ptr(), out["hit_eos"].data_ptr(),
        stream_ptr(dev)))


TOP_MAX = 32  # alternatives of a position that token_logprobs returns at most


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, logprob: torch.Tensor, entropy: torch.Tensor,
                   top_logprob: Optional[torch.Tensor] = None, top_token: Optional[torch.Tensor] = None) -> None:
    """Log probabilities of ``tokens`` under ``logits``, the entropy and the best alternatives
    (``yapd_token_logprobs``), into caller tensors.

    ``logits`` is bf16 or fp32 ``[n, V]`` or ``[rows, bl, V]`` with a unit last stride (any others);
    ``tokens`` (int64), ``logprob`` and ``entropy`` (fp32) have its leading shape, ``top_logprob``
    (fp32) and ``top_token`` (int64) ``[..., k]`` with ``0 <= k <= 32``.  A token below 0 marks a position
    without one (log probability 0), one past the vocabulary gives NaN."""
    dev = logits.device
    if logits.is_cuda and dev.index != torch.cuda.current_device():
        with torch.cuda.device(dev):  # the launch goes to the current device
            return token_logprobs(logits, tokens, logprob, entropy, top_logprob, top_token)
    check_token_logprobs(logits, tokens)
    lead = logits.shape[:-1]
    require_cuda(logprob, "logprob", torch.float32, dev)
    require_cuda(entropy, "entropy", torch.float32, dev)
    require(logprob.shape == lead and entropy.shape == lead, "logprob and entropy must have the logits' leading shape")
    k = 0
    if top_logprob is not None or top_token is not None:
        require(top_logprob is not None and top_token is not None, "top_logprob and top_token come together")
        require_cuda(top_logprob, "top_logprob", torch.float32, dev)
        require_cuda(top_token, "top_token", torch.int64, dev)
        k = top_token.shape[-1]
        require(top_logprob.shape == top_token.shape and top_token.shape[:-1] == lead,
                "top_logprob and top_token must be [..., k] on the logits' leading shape")
    launch_token_logprobs(logits, tokens, k, logprob, entropy, top_logprob, top_token)


def check_token_logprobs(logits: torch.Tensor, tokens: torch.Tensor) -> None:
    dev, shape = logits.device, logits.shape
    require_cuda(logits, "logits", torch.float32 if logits.dtype == torch.float32 else torch.bfloat16, dev,
                 contiguous=False)
    require(len(shape) in (2, 3) and (shape[-1] <= 1 or logits.stride(-1) == 1),
            "logits must be [n, V] or [rows, bl, V] with unit last stride")
    require_cuda(tokens, "tokens", torch.int64, dev)
    require(tokens.shape == shape[:-1], "tokens must have the logits' leading shape")


def launch_token_logprobs(logits, tokens, k: int, logprob, entropy, top_logprob, top_token) -> None:
    """:func:`token_logprobs` on tensors that are known to fit."""
    shape, stride = logits.shape, logits.stride()
    if len(shape) == 2:
        seq, pos, rows, bl = stride[0], 0, shape[0], 1
    else:
        (seq, pos, _), (rows, bl, _) = stride, shape
    check(load_library().yapd_token_logprobs(
        logits.data_ptr(), logits.dtype == torch.float32, seq, pos, rows, bl, shape[-1], tokens.data_ptr(), k,
        logprob.data_ptr(), entropy.data_ptr(), ptr(top_logprob), ptr(top_token), stream_ptr(logits.device)))


def sample_tokens(logits: torch.Tensor, uniform: torch.Tensor, token: torch.Tensor, logprob: torch.Tensor, *,
                  temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) -> None:
    """A token drawn from every row of ``logits`` with the random number ``uniform`` (``yapd_sample_tokens``), into
    caller tensors that share no memory with the inputs; see :func:`yapd_amd.scoring.sample_tokens`."""
    dev = logits.device
    if elsewhere(logits):
        with torch.cuda.device(dev):  # the launch goes to the current device
            return sample_tokens(logits, uniform, token, logprob, temperature=temperature, top_k=top_k, top_p=top_p,
                                 min_p=min_p)
    f32, shape, stride = torch.float32, logits.shape, logits.stride()
    wide = logits.dtype is f32
    require_cuda(logits, "logits", f32 if wide else torch.bfloat16, dev, contiguous=False)
    require(len(shape) in (2, 3) and (shape[-1] <= 1 or stride[-1] == 1),
            "logits must be [n, V] or [rows, bl, V] with unit last stride")
    lead = shape[:-1]

    def setting(name, t, dtype):
        """(address or None, number) of a setting."""
        if not isinstance(t, torch.Tensor):
            return None, t
        require_cuda(t, name, dtype, dev)
        if t.shape != lead:
            raise ValueError(f"{name} must have the logits' leading shape")
        return t.data_ptr(), 0

    for name, t, dtype in (("uniform", uniform, f32), ("token", token, torch.int64), ("logprob", logprob, f32)):
        if not isinstance(t, torch.Tensor):
            raise ValueError(f"{name} must be a tensor")
        require_cuda(t, name, dtype, dev)
        if t.shape != lead:
            raise ValueError(f"{name} must have the logits' leading shape")
    t, t_all = setting("temperature", temperature, f32)
    k, k_all = setting("top_k", top_k, torch.int32)
    p, p_all = setting("top_p", top_p, f32)
    m, m_all = setting("min_p", min_p, f32)
    require(k_all == int(k_all), "top_k must be an integer")
    rows, bl = (shape[0], 1) if len(shape) == 2 else lead
    check(load_library().yapd_sample_tokens(
        logits.data_ptr(), wide, stride[0], 0 if len(shape) == 2 else stride[1], rows, bl, shape[-1], uniform.data_ptr(), t,
        t_all, k, max(min(int(k_all), 2**31 - 1), 0), p, p_all, m, m_all, token.data_ptr(), logprob.data_ptr(),
        stream_ptr(dev)))


# --------------------------------------------------------------------------- #
# (a) paged block attention
# --------------------------------------------------------------------------- #

def attn_plan(kv_len, target_items: int = 192, min_split_keys: int = 1024):
    """Host planner: ``(work [n,4] int32, merge [m,3] int32, n_slots)`` numpy arrays.

    Rows are cut into work items of whole 32-key chunks so that about
    ``target_items`` items exist (192 is roughly how many four-head work items
    the MI355X keeps in flight, so only rows longer than the average share are
    split), never into items shorter than ``min_split_keys``; items are ordered
    longest first.  1024 keys (1 MB of K/V per four-head item) is where the
    split rows' merges and per-item start-up cost less than the tail they
    remove: on 256 rows of log-uniform [64, 2048] keys, 1024 runs 125 us per
    layer against 128 us at 128 keys and 131 us at 1280 keys.
    """
    import numpy as np
    kv = np.ascontiguousarray(np.asarray(kv_len, dtype=np.int32))
    rows = int(kv.size)
    unit = 32
    cap = int(sum((int(x) + unit - 1) // unit for x in kv)) + rows
    work = np.zeros((cap, 4), dtype=np.int32)
    merge = np.zeros((rows, 3), dtype=np.int32)
    nw, nm, ns = ctypes.c_int(), ctypes.c_int(), ctypes.c_int()
    check(load_library().yapd_attn_plan(
        kv.ctypes.data, rows, int(target_items), int(min_split_keys), work.ctypes.data, cap,
        merge.ctypes.data, rows, ctypes.byref(nw), ctypes.byref(nm), ctypes.byref(ns)))
    return work[: nw.value].copy(), merge[: nm.value].copy(), ns.value


def attn_paged_block(q: torch.Tensor, pool: torch.Tensor, table: torch.Tensor, kv_len: torch.Tensor,
                     work: torch.Tensor, merge: Optional[torch.Tensor], part_o: Optional[torch.Tensor],
                     part_ml: Optional[torch.Tensor], out: torch.Tensor, scale: float,
                     causal: bool = False) -> None:
    """``out [rows, bl, H, 64] = softmax(q K^T * scale) V`` over each row's pages.

    ``causal``: query ``i`` of the block sees keys ``< kv_len - bl + i + 1`` (prefill).
    """
    dev = q.device
    require_cuda(q, "q", torch.bfloat16, dev)
    require(q.dim() == 4 and q.shape[3] == 64, "q must be [rows, bl, H, 64]")
    rows, bl, H, _ = q.shape
    require_cuda(pool, "pool", torch.bfloat16, dev)
    require(pool.dim() == 4 and pool.shape[1] == 2 and pool.shape[2] == H and pool.shape[3] == 1024,
            "pool must be [pages, 2, H, 16*64]")
    require_cuda(table, "table", torch.int32, dev, contiguous=False)
    require(table.dim() == 2 and table.shape[0] >= rows and table.stride(1) == 1,
            "table must be [>= rows, max_pages] with unit column stride")
    require_cuda(kv_len, "kv_len", torch.int32, dev)
    require(kv_len.numel() >= rows, "kv_len must have rows entries")
    require_cuda(work, "work", torch.int32, dev)
    require(work.dim() == 2 and work.shape[1] == 4, "work must be [n, 4]")
    n_merge = 0 if merge is None else int(merge.shape[0])
    n_slots = 0
    if n_merge:
        require_cuda(merge, "merge", torch.int32, dev)
        require_cuda(part_o, "part_o", torch.float32, dev)
        require_cuda(part_ml, "part_ml", torch.float32, dev)
        n_slots = int(part_o.shape[0])
        require(tuple(part_o.shape[1:]) == (bl, H, 64) and tuple(part_ml.shape) == (n_slots, bl, H, 2),
                "part_o/part_ml shapes")
    require_cuda(out, "out", torch.bfloat16, dev)
    require(tuple(out.shape) == (rows, bl, H, 64), "out must match q")
    check(load_library().yapd_attn_paged_block(
        q.data_ptr(), pool.data_ptr(), pool.shape[0], table.data_ptr(), table.stride(0), table.shape[1],
        kv_len.data_ptr(),
        rows, bl, H, work.data_ptr(), int(work.shape[0]), ptr(merge), n_merge, None, ptr(part_o), ptr(part_ml),
        n_slots, float(scale), int(bool(causal)), out.data_ptr(), stream_ptr(dev)))


WINDOW_CAP = 2**30  # windows, sinks and lengths from here on are taken as this


def attn_window(q: torch.Tensor, pool: torch.Tensor, table: torch.Tensor, kv_len: torch.Tensor, out: torch.Tensor,
                scale: float, *, window: int, sinks: int = 0, causal: bool = True,
                q_start: Optional[torch.Tensor] = None, max_q: Optional[int] = None, max_kv: Optional[int] = None,
                workspace: Optional[torch.Tensor] = None) -> None:
    """``out = softmax(q K^T * scale) V`` over each row's pages with a sliding window and sink tokens.

    Query ``i`` of a row with ``n`` queries stands at position ``p = kv_len - n + i`` and sees key
    ``j`` iff ``j < hi`` and (``j < sinks`` or ``j > p - window``), with ``hi = p + 1`` (``causal``) or
    ``kv_len`` (a block step).  Queries are ``[rows, bl, H, 64]``, or packed ``[n_q, H, 64]`` with the
    device ``q_start [rows + 1]`` (int32, not decreasing): row ``r`` has rows ``q_start[r]`` up to
    ``q_start[r + 1]`` of ``q`` and ``out``; of more than ``max_q`` the first ``max_q`` are computed, at the positions
    that the whole row gives them.  Rows of ``out`` that are not computed or belong to no row are left as they were.  ``q`` may be a view with packed heads and any token stride (a slice of
    a fused QKV buffer); ``out`` is contiguous; one that shares memory with ``q`` or the pool is refused.

    Lengths are read on the device: no plan, and a captured call follows them.  ``max_q`` and
    ``max_kv`` are the host's upper bounds (default: all queries, all positions the table maps).
    ``scale`` is positive, and scores have to stay below 2^30 in magnitude.
    Few queries over many keys need a float32 ``workspace``
    (``yapd_attn_window_workspace``), allocated here unless given.
    """
    dev = q.device
    if q.is_cuda and dev.index != torch.cuda.current_device():
        with torch.cuda.device(dev):  # the launch goes to the current device
            return attn_window(q, pool, table, kv_len, out, scale, window=window, sinks=sinks, causal=causal,
                               q_start=q_start, max_q=max_q, max_kv=max_kv, workspace=workspace)
    bf16, i32 = torch.bfloat16, torch.int32
    require_cuda(q, "q", bf16, dev, contiguous=False)
    # sizes and strides are asked for once: a single token's call is host time
    shape, stride = q.shape, q.stride()
    dims = len(shape)
    require((dims >= 2 and stride[-1] == 1 and stride[-2] == 64) or q.numel() == 0, "q's heads must be packed")
    packed = q_start is not None
    if packed:
        require(dims == 3 and shape[2] == 64, "packed q must be [n_q, H, 64]")
        n_q, H, _ = shape
        require_cuda(q_start, "q_start", i32, dev)
        rows = q_start.numel() - 1
        require(rows >= 0, "q_start must be [rows + 1]")
        if max_q is None:
            max_q = n_q
        require(n_q == 0 or rows == 0 or max_q >= 1, "max_q must be >= 1")
        tok = stride[0] if n_q > 1 else H * 64
    else:
        require(dims == 4 and shape[3] == 64, "q must be [rows, bl, H, 64] (or [n_q, H, 64] with q_start)")
        rows, bl, H, _ = shape
        n_q = rows * bl
        require(max_q is None or max_q == bl, "max_q is given by q's shape unless q is packed")
        max_q = bl
        tok = stride[1] if bl > 1 else stride[0] if rows > 1 else H * 64
        require(rows <= 1 or stride[0] == bl * tok or n_q == 0, "q's rows must follow each other")
    require_cuda(pool, "pool", bf16, dev)
    pool_shape = pool.shape
    if pool_shape[1:] != (2, H, 1024):
        raise ValueError("pool must be [pages, 2, H, 16*64]")
    require_cuda(table, "table", i32, dev, contiguous=False)
    table_shape, table_stride = table.shape, table.stride()
    require(len(table_shape) == 2 and table_shape[0] >= rows and (table_shape[1] == 1 or table_stride[1] == 1),
            "table must be [>= rows, max_pages] with unit column stride")
    cols, pitch = table_shape[1], table_stride[0]
    require(rows <= 1 or pitch >= cols, "table rows must not overlap")
    require_cuda(kv_len, "kv_len", i32, dev)
    require(kv_len.numel() >= rows, "kv_len must have rows entries")
    require_cuda(out, "out", bf16, dev)
    require(out.shape == shape, "out must match q")
    require(window >= 1 and sinks >= 0, "need window >= 1 and sinks >= 0")
    if n_q == 0 or rows == 0:
        return
    require(cols >= 1, "the table maps no page")
    window, sinks = min(int(window), WINDOW_CAP), min(int(sinks), WINDOW_CAP)
    kv_max = cols * 16 if max_kv is None else min(int(max_kv), cols * 16)
    require(kv_max >= 1, "max_kv must be >= 1")
    max_q = min(int(max_q), n_q)
    lib = load_library()
    need = lib.yapd_attn_window_workspace(rows, max_q, n_q, packed, H, window, sinks, kv_max)
    if need > 0 and workspace is None:
        workspace = torch.empty(need, dtype=torch.float32, device=dev)
    if workspace is not None:
        require_cuda(workspace, "workspace", torch.float32, dev)
    check(lib.yapd_attn_window(
        q.data_ptr(), tok, pool.data_ptr(), pool_shape[0], table.data_ptr(), max(pitch, cols), cols,
        kv_len.data_ptr(), ptr(q_start), rows, max_q, n_q, H, window, sinks, causal, kv_max, scale, ptr(workspace),
        0 if workspace is None else workspace.numel(), out.data_ptr(), stream_ptr(dev)))


def kv_write(k: torch.Tensor, v: torch.Tensor, pool: torch.Tensor, table: torch.Tensor,
             pos0: torch.Tensor, bl: int) -> None:
    """Scatter ``k, v`` (``[rows*bl, H, 64]`` views, unit last strides) into the pages."""
    dev = k.device
    for name, t in (("k", k), ("v", v)):
        require_cuda(t, name, torch.bfloat16, dev, contiguous=False)
        require(t.dim() == 3 and t.shape[2] == 64 and t.stride(2) == 1 and t.stride(1) == 64,
                f"{name} must be [tokens, H, 64] with packed heads")
    H = k.shape[1]
    require_cuda(pool, "pool", torch.bfloat16, dev)
    require(pool.dim() == 4 and pool.shape[2] == H and pool.shape[3] == 1024, "pool must be [pages, 2, H, 1024]")
    require_cuda(table, "table", torch.int32, dev)
    require_cuda(pos0, "pos0", torch.int32, dev)
    rows = int(pos0.numel())
    require(k.shape[0] == rows * bl and v.shape[0] == rows * bl, "k/v must hold rows*bl tokens")
    check(load_library().yapd_kv_write(
        k.data_ptr(), v.data_ptr(), k.stride(0), v.stride(0), pool.data_ptr(), pool.shape[0],
        table.data_ptr(), table.stride(0), table.shape[1], pos0.data_ptr(), rows, bl, H, stream_ptr(dev)))


def kv_gather(pool: torch.Tensor, table_row: torch.Tensor, kv_len: int):
    """Dense ``K, V [kv_len, H, 64]`` of one row (page-table gather, debug/test path)."""
    dev = pool.device
    require_cuda(pool, "pool", torch.bfloat16, dev)
    require_cuda(table_row, "table_row", torch.int32, dev)
    H = pool.shape[2]
    require(table_row.numel() * 16 >= kv_len, "table_row too short for kv_len")
    k = torch.empty(kv_len, H, 64, dtype=torch.bfloat16, device=dev)
    v = torch.empty_like(k)
    check(load_library().yapd_kv_gather(pool.data_ptr(), pool.shape[0], table_row.data_ptr(), table_row.numel(),
                                        int(kv_len), H, k.data_ptr(), v.data_ptr(), stream_ptr(dev)))
    return k, v


def pool_pointers(pools):
    """The device addresses of every layer's pool, and the pools' common shape and device, checked.

    Pools are bf16, or uint8 for an 8-bit cache (``shape[3]`` tells which)."""
    require(len(pools) >= 1, "no pools")
    shape, dev = pools[0].shape, pools[0].device
    dtype = torch.uint8 if pools[0].dtype is torch.uint8 else torch.bfloat16
    index = pools[0].get_device()
    ptrs = []
    for p in pools:
        if p.dtype is not dtype or p.shape != shape or p.get_device() != index or not p.is_contiguous():
            require_cuda(p, "pool", dtype, dev)
            raise ValueError("every layer's pool must have the same shape")
        ptrs.append(p.data_ptr())
    require_cuda(pools[0], "pool", dtype, dev)
    require(len(shape) == 4 and shape[0] >= 1 and shape[1] == 2 and shape[3] == (TILE8 if dtype is torch.uint8 else 1024),
            "pools must be [pages, 2, H, 16*64] (uint8: [pages, 2, H, 16*64 + 16])")
    return array("Q", ptrs), shape, dev


def page_ids(ids, name: str):
    """Host page ids (a sequence of integers or an integer array) as int32."""
    import numpy as np
    if isinstance(ids, torch.Tensor):
        require(not ids.is_cuda, f"{name} must be host integers, not a GPU tensor")
        ids = ids.numpy()
    a = np.asarray(ids)
    if a.dtype != np.int32:  # the library checks the range of those that are
        require(a.size == 0 or (a.dtype.kind in "iu" and bool((a >= 0).all()) and bool((a < 2**31).all())),
                f"{name} must be page ids (integers of [0, 2^31))")
        a = a.astype(np.int32)
    require(a.ndim == 1, f"{name} must be one-dimensional")
    return np.ascontiguousarray(a)


def check_page_pairs(src, dst, n_pages: int) -> None:
    """What ``yapd_kv_copy_pages`` refuses of page ids, for pools on the CPU."""
    import numpy as np
    require(src.size == dst.size, "src and dst must have the same length")
    both = np.concatenate([src, dst])
    require(not both.size or (both.min() >= 0 and both.max() < n_pages), f"pairs outside the pool's {n_pages} pages")
    require(np.unique(dst).size == dst.size, "a page is the destination of two pairs")
    require(not np.intersect1d(src, dst).size, "a page is a source and a destination")


def kv_copy_pages(pools, src, dst) -> None:
    """``pool[dst[i]] = pool[src[i]]`` for every pair ``i`` in every layer's pool of ``pools``, in one
    launch (per 64 layers and 384 pairs).

    ``src`` and ``dst`` are host page ids.  A source may repeat (a fork); a page that is the
    destination of two pairs, or a source and a destination, is refused, so the result does not
    depend on the order of the copies."""
    ptrs, shape, dev = pool_pointers(pools)
    if dev.index != torch.cuda.current_device():
        with torch.cuda.device(dev):  # the launch goes to the current device
            return kv_copy_pages(pools, src, dst)
    src, dst = page_ids(src, "src"), page_ids(dst, "dst")
    require(src.size == dst.size, "src and dst must have the same length")
    copy = load_library().yapd_kv_copy_pages if shape[3] == 1024 else load_library().yapd_kv8_copy_pages
    check(copy(ptrs.buffer_info()[0], len(ptrs), shape[0], shape[2], src.ctypes.data, dst.ctypes.data, src.size,
               stream_ptr(dev)))


# --------------------------------------------------------------------------- #
# drafted tokens: the 8-bit cache, attention for trees, the accepted tokens
# --------------------------------------------------------------------------- #

TILE8 = 16 * 64 + 16  # bytes of one head's plane on a page of an 8-bit pool: codes, then a scale byte a token
MAX_NODES = 64        # nodes of a drafted tree: bits of a mask


def elsewhere(t: torch.Tensor) -> bool:
    """Whether ``t`` is on another GPU than the current one, to which launches go."""
    return t.is_cuda and t.get_device() != torch._C._cuda_getDevice()


def kv_bits(pool: torch.Tensor) -> int:
    """8 or 16: the width of a pool's values."""
    return 8 if pool.dtype is torch.uint8 else 16


def check_pool(pool: torch.Tensor, name: str, dtype: torch.dtype, dev: torch.device, heads: int) -> None:
    require_cuda(pool, name, dtype, dev)
    tile = TILE8 if dtype is torch.uint8 else 1024
    if pool.shape[1:] != (2, heads, tile):
        raise ValueError(f"{name} must be [pages, 2, {heads}, {'16*64 + 16' if tile == TILE8 else '16*64'}]")


def check_table(table: torch.Tensor, name: str, dev: torch.device, rows: int):
    """``(columns, row pitch)`` of an int32 page table of at least ``rows`` rows."""
    require_cuda(table, name, torch.int32, dev, contiguous=False)
    shape, stride = table.shape, table.stride()
    if len(shape) != 2 or shape[0] < rows or shape[1] < 1 or (shape[1] != 1 and stride[1] != 1):
        raise ValueError(f"{name} must be [>= rows, max_pages] with unit column stride")
    if rows > 1 and stride[0] < shape[1]:
        raise ValueError(f"{name}'s rows must not overlap")
    return shape[1], max(stride[0], shape[1])


def kv8_write(k: torch.Tensor, v: torch.Tensor, pool: torch.Tensor, table: torch.Tensor, pos0: torch.Tensor, *,
              q_start: Optional[torch.Tensor] = None) -> None:
    """Quantise fresh ``k, v`` (bf16 ``[tokens, H, 64]`` with packed heads, any token stride) into the pages of an
    8-bit pool (``yapd_kv8_write``): uint8 ``[pages, 2, H, 16*64 + 16]``, one power-of-two scale a (token, head, plane).

    Row ``r``'s tokens go to positions ``pos0[r], pos0[r] + 1, ...``: ``tokens / rows`` of them each (``rows`` the entries
    of ``pos0``), or packed ``[q_start[r], q_start[r + 1])`` (int32, not decreasing).  Positions that the table does not
    map to a page of the pool are left out; every other byte of the pool stays.  NaN is written as 0, infinities as
    the largest finite value.  The positions written must belong to one row alone: two tokens of one position may leave
    the codes of one and the scale of the other."""
    dev = k.device
    if elsewhere(k):
        with torch.cuda.device(dev):  # the launch goes to the current device
            return kv8_write(k, v, pool, table, pos0, q_start=q_start)
    for name, t in (("k", k), ("v", v)):
        require_cuda(t, name, torch.bfloat16, dev, contiguous=False)
    shape, k_stride, v_stride = k.shape, k.stride(), v.stride()
    require(len(shape) == 3 and shape == v.shape and shape[2] == 64, "k and v must be [tokens, H, 64]")
    n, H, _ = shape
    require(n * H == 0 or (k_stride[2] == v_stride[2] == 1 and (H == 1 or k_stride[1] == v_stride[1] == 64)),
            "k's and v's heads must be packed")
    check_pool(pool, "pool", torch.uint8, dev, H)
    require_cuda(pos0, "pos0", torch.int32, dev)
    rows = pos0.numel()
    cols, pitch = check_table(table, "table", dev, rows)
    if q_start is None:
        require(n % rows == 0 if rows else n == 0, "k and v must hold the same number of tokens for every row")
    else:
        require_cuda(q_start, "q_start", torch.int32, dev)
        require(q_start.numel() == rows + 1, "q_start must be [rows + 1]")
    if n == 0 or rows == 0:
        return
    k_tok, v_tok = (k_stride[0], v_stride[0]) if n > 1 else (H * 64, H * 64)
    check(load_library().yapd_kv8_write(
        k.data_ptr(), v.data_ptr(), k_tok, v_tok, pool.data_ptr(), pool.shape[0], table.data_ptr(), pitch, cols,
        pos0.data_ptr(), ptr(q_start), rows, n, H, stream_ptr(dev)))


def kv8_unpack(pool8: torch.Tensor, table8: torch.Tensor, kv_len: torch.Tensor, pool: torch.Tensor,
               table: torch.Tensor, *, max_kv: Optional[int] = None) -> None:
    """Read an 8-bit cache back: the pages that hold positions ``[0, kv_len[r])`` of every row, mapped by ``table8``
    in ``pool8``, become the bf16 pages of ``pool`` that ``table`` maps there (``yapd_kv8_unpack``).  Exact: a code
    times its scale is a bf16 value.  A page's slots past ``kv_len`` are converted as they stand.

    ``kv_len`` is read on the device; ``max_kv`` is the host's upper bound (default: all that both tables map),
    past which nothing is converted.  Columns that either table does not map to a page of its pool are left out.  A page
    of ``pool`` that two pages of ``pool8`` go to may hold some of each."""
    dev = pool8.device
    if elsewhere(pool8):
        with torch.cuda.device(dev):  # the launch goes to the current device
            return kv8_unpack(pool8, table8, kv_len, pool, table, max_kv=max_kv)
    require(pool8.dim() == 4, "pool8 must be [pages, 2, H, 16*64 + 16]")
    H = pool8.shape[2]
    check_pool(pool8, "pool8", torch.uint8, dev, H)
    check_pool(pool, "pool", torch.bfloat16, dev, H)
    require_cuda(kv_len, "kv_len", torch.int32, dev)
    rows = kv_len.numel()
    if rows == 0:
        return
    cols8, pitch8 = check_table(table8, "table8", dev, rows)
    cols, pitch = check_table(table, "table", dev, rows)
    most = min(cols8, cols) * 16
    most = most if max_kv is None else min(int(max_kv), most)
    require(most >= 1, "max_kv must be >= 1")
    check(load_library().yapd_kv8_unpack(
        pool8.data_ptr(), pool8.shape[0], table8.data_ptr(), pitch8, cols8, kv_len.data_ptr(), rows, most, H,
        pool.data_ptr(), pool.shape[0], table.data_ptr(), pitch, cols, stream_ptr(dev)))


def tree_masks(parents):
    """The masks of one drafted tree for :func:`attn_tree`, as an int64 numpy array: node ``i`` sees itself and its
    ancestors.  ``parents[i]`` is the node that ``i`` follows (an earlier one), or -1 for the row's last token."""
    import numpy as np
    parents = [int(p) for p in parents]
    require(len(parents) <= MAX_NODES, f"a tree has at most {MAX_NODES} nodes")
    masks = []
    for i, p in enumerate(parents):
        require(-1 <= p < i, "a node's parent must be an earlier node, or -1")
        masks.append((masks[p] if p >= 0 else 0) | 1 << i)
    return np.array(masks, dtype=np.uint64).view(np.int64)


def attn_tree(q: torch.Tensor, pool: torch.Tensor, table: torch.Tensor, kv_len: torch.Tensor, mask: torch.Tensor,
              out: torch.Tensor, scale: float, *, window: Optional[int] = None, sinks: int = 0,
              q_start: Optional[torch.Tensor] = None, max_q: Optional[int] = None, max_kv: Optional[int] = None,
              workspace: Optional[torch.Tensor] = None) -> None:
    """``out = softmax(q K^T * scale) V`` for trees of at most 64 drafted tokens over each row's pages, bf16 or 8-bit.

    A row's ``n`` nodes are its last positions, ``ctx = kv_len - n`` up to ``kv_len``, their keys already in the cache.
    Node ``i`` sees node ``j`` iff bit ``j`` of its ``mask`` (int64) is set (:func:`tree_masks`), and key ``j < ctx`` iff
    ``j < sinks`` or ``j > ctx + depth - window``, ``depth`` the number of other nodes in its mask.  With one node and
    mask 1 that is the next token of an ordinary decode.  A node that sees nothing gets zeros.

    Nodes are ``[rows, n, H, 64]`` (``mask [rows, n]``), or packed ``[n_q, H, 64]`` (``mask [n_q]``) with the device
    ``q_start [rows + 1]`` (int32, not decreasing); of a row of more than ``max_q`` nodes the first ``max_q`` are computed, as
    the row's first.  Rows of ``out`` that are not computed or belong to no row are left as they were.  ``q`` may be a
    view with packed heads and any token stride; ``out`` is contiguous; one that shares memory with ``q`` or the pool is refused.

    Lengths and masks are read on the device: a captured call follows them.  ``max_q`` (default: all, at most 64) and
    ``max_kv`` (default: all positions the table maps) are the host's upper bounds; ``window`` (default: none) is at least
    ``n``, of packed nodes at least 1.  Scores have to stay below 2^30 in magnitude.  Few nodes over many keys need a
    float32 ``workspace`` (``yapd_attn_tree_workspace``), allocated here unless given."""
    dev = q.device
    if elsewhere(q):
        with torch.cuda.device(dev):  # the launch goes to the current device
            return attn_tree(q, pool, table, kv_len, mask, out, scale, window=window, sinks=sinks, q_start=q_start,
                             max_q=max_q, max_kv=max_kv, workspace=workspace)
    bf16, i32 = torch.bfloat16, torch.int32
    require_cuda(q, "q", bf16, dev, contiguous=False)
    # sizes and strides are asked for once, and messages made only for what fails: a single token's call is host time
    shape, stride = q.shape, q.stride()
    if q_start is not None:
        require(len(shape) == 3 and shape[2] == 64, "packed q must be [n_q, H, 64]")
        n_q, H, _ = shape
        require_cuda(q_start, "q_start", i32, dev)
        rows = q_start.numel() - 1
        require(rows >= 0, "q_start must be [rows + 1]")
        max_q = min(n_q, MAX_NODES) if max_q is None else int(max_q)
        require(n_q == 0 or rows == 0 or max_q >= 1, "max_q must be >= 1")
        tok = stride[0] if n_q > 1 else H * 64
    else:
        require(len(shape) == 4 and shape[3] == 64, "q must be [rows, n, H, 64] (or [n_q, H, 64] with q_start)")
        rows, bl, H, _ = shape
        n_q = rows * bl
        require(max_q is None or max_q == bl, "max_q is given by q's shape unless q is packed")
        max_q = bl
        tok = stride[1] if bl > 1 else stride[0] if rows > 1 else H * 64
        require(rows <= 1 or stride[0] == bl * tok or n_q == 0, "q's rows must follow each other")
    require(n_q * H == 0 or (stride[-1] == 1 and (H == 1 or stride[-2] == 64)), "q's heads must be packed")
    bits = kv_bits(pool)
    check_pool(pool, "pool", torch.uint8 if bits == 8 else bf16, dev, H)
    require_cuda(mask, "mask", torch.int64, dev)
    require_cuda(kv_len, "kv_len", i32, dev)
    require_cuda(out, "out", bf16, dev)
    if mask.shape != shape[:-2] or out.shape != shape or kv_len.numel() < rows:
        require(mask.shape == shape[:-2], "mask must be q's shape without heads")
        require(out.shape == shape, "out must match q")
        raise ValueError("kv_len must have rows entries")
    window = WINDOW_CAP if window is None else min(int(window), WINDOW_CAP)
    sinks = min(int(sinks), WINDOW_CAP)
    require(window >= 1 and sinks >= 0, "need window >= 1 and sinks >= 0")
    if n_q == 0 or rows == 0:
        return
    cols, pitch = check_table(table, "table", dev, rows)
    kv_max = cols * 16 if max_kv is None else min(int(max_kv), cols * 16)
    max_q = min(max_q, n_q)
    lib = load_library()
    floats = 0
    if workspace is None:
        floats = lib.yapd_attn_tree_workspace(rows, max_q, n_q, H, window if q_start is None else max(window, max_q), sinks,
                                              kv_max, bits)
        if floats > 0:
            workspace = torch.empty(floats, dtype=torch.float32, device=dev)
    else:
        require_cuda(workspace, "workspace", torch.float32, dev)
        floats = workspace.numel()
    check(lib.yapd_attn_tree(
        q.data_ptr(), tok, pool.data_ptr(), bits, pool.shape[0], table.data_ptr(), pitch, cols, kv_len.data_ptr(),
        None if q_start is None else q_start.data_ptr(), mask.data_ptr(), rows, max_q, n_q, H, window, sinks, kv_max, scale,
        None if workspace is None else workspace.data_ptr(), floats, out.data_ptr(), stream_ptr(dev)))


def kv_keep(pools, table: torch.Tensor, base: torch.Tensor, kept: torch.Tensor, n_kept: torch.Tensor) -> None:
    """Move the accepted nodes of drafted trees together, in every layer's pool of ``pools`` (bf16 or 8-bit):
    position ``base[r] + i`` of row ``r`` becomes what position ``base[r] + kept[r, i]`` was, for ``i < n_kept[r]``, in one
    launch per 64 layers (``yapd_kv_keep``).

    ``base [rows]``, ``kept [rows, m]`` (``m <= 64``) and ``n_kept [rows]`` are device int32, so a verification on the
    device needs no synchronisation.  A row's values are all read before the first is written: any nodes in any
    order.  Positions that the table does not map to a page of the pool are left out (page 0 is one, also where a table names
    it for positions that hold nothing).  The written pages must belong to one row alone."""
    ptrs, shape, dev = pool_pointers(pools)
    if elsewhere(pools[0]):
        with torch.cuda.device(dev):  # the launch goes to the current device
            return kv_keep(pools, table, base, kept, n_kept)
    i32 = torch.int32
    require_cuda(base, "base", i32, dev)
    require_cuda(kept, "kept", i32, dev, contiguous=False)
    require_cuda(n_kept, "n_kept", i32, dev)
    rows = base.numel()
    shape_k, stride_k = kept.shape, kept.stride()
    if not (len(shape_k) == 2 and shape_k[0] == rows and shape_k[1] <= MAX_NODES and (shape_k[1] <= 1 or stride_k[1] == 1)
            and (rows <= 1 or stride_k[0] >= shape_k[1])):
        raise ValueError(f"kept must be [rows, at most {MAX_NODES}] with unit column stride")
    require(n_kept.numel() == rows, "n_kept must have rows entries")
    cols, pitch = check_table(table, "table", dev, rows)
    if rows == 0 or shape_k[1] == 0:
        return
    check(load_library().yapd_kv_keep(
        ptrs.buffer_info()[0], len(ptrs), 16 if shape[3] == 1024 else 8, shape[0], shape[2], table.data_ptr(), pitch, cols,
        base.data_ptr(), kept.data_ptr(), max(stride_k[0], shape_k[1]), shape_k[1], n_kept.data_ptr(), rows, stream_ptr(dev)))


# --------------------------------------------------------------------------- #
# (b) GEMMs and norms
# --------------------------------------------------------------------------- #

def _mat(t: torch.Tensor, name: str, dev) -> None:
    require_cuda(t, name, torch.bfloat16, dev, contiguous=False)
    if not (t.dim() == 2 and t.stride(1) == 1):
        raise ValueError(f"{name} must be a 2-D row-major view")


def gemm_bf16(A: torch.Tensor, W: torch.Tensor, out: torch.Tensor) -> None:
    """``out[M, N] = A[M, K] @ W[N, K]^T`` in bf16 with fp32 accumulation."""
    dev = A.device
    _mat(A, "A", dev)
    _mat(W, "W", dev)
    _mat(out, "out", dev)
    M, K = A.shape
    N = W.shape[0]
    require(W.shape[1] == K and tuple(out.shape) == (M, N), "gemm shapes")
    check(load_library().yapd_gemm_bf16(A.data_ptr(), A.stride(0), W.data_ptr(), W.stride(0), M, N, K,
                                        out.data_ptr(), out.stride(0), stream_ptr(dev)))


def gemm_bf16_residual(A: torch.Tensor, W: torch.Tensor, residual: torch.Tensor) -> None:
    """``residual = bf16(residual + bf16(A @ W^T))`` in place (projection + residual add)."""
    dev = A.device
    _mat(A, "A", dev)
    _mat(W, "W", dev)
    _mat(residual, "residual", dev)
    M, K = A.shape
    N = W.shape[0]
    require(W.shape[1] == K and tuple(residual.shape) == (M, N), "gemm shapes")
    check(load_library().yapd_gemm_bf16_residual(A.data_ptr(), A.stride(0), W.data_ptr(), W.stride(0), M, N, K,
                                                 residual.data_ptr(), residual.stride(0), stream_ptr(dev)))


def gemm_head_shift(hidden: torch.Tensor, shift_ctx: torch.Tensor, W: torch.Tensor, logits: torch.Tensor) -> None:
    """Token-shifted head: ``logits[r, j] = W @ (j ? hidden[r, j-1] : shift_ctx[r])``.

    ``hidden [rows, bl, D]`` contiguous, ``shift_ctx [rows, 1, D]`` contiguous,
    ``logits [rows, bl, V]`` with a unit last stride (padded pitch allowed).
    """
    dev = hidden.device
    require_cuda(hidden, "hidden", torch.bfloat16, dev)
    require_cuda(shift_ctx, "shift_ctx", torch.bfloat16, dev)
    _mat(W, "W", dev)
    rows, bl, D = hidden.shape
    require(tuple(shift_ctx.shape) == (rows, 1, D), "shift_ctx must be [rows, 1, D]")
    require_cuda(logits, "logits", torch.bfloat16, dev, contiguous=False)
    V = W.shape[0]
    require(tuple(logits.shape) == (rows, bl, V) and logits.stride(2) == 1 and logits.stride(0) == bl * logits.stride(1),
            "logits must be [rows, bl, V] with rows packed")
    check(load_library().yapd_gemm_head_shift(hidden.data_ptr(), shift_ctx.data_ptr(), rows, bl, D, W.data_ptr(),
                                              W.stride(0), V, logits.data_ptr(), logits.stride(1), stream_ptr(dev)))


def gemm_swiglu(A: torch.Tensor, W_gu_interleaved: torch.Tensor, act: torch.Tensor) -> None:
    """``act[M, F] = silu(A Wg^T) * (A Wu^T)`` with gate/up rows interleaved per 32 (see interleave_gate_up)."""
    dev = A.device
    _mat(A, "A", dev)
    require_cuda(W_gu_interleaved, "W_gu", torch.bfloat16, dev)
    _mat(act, "act", dev)
    M, K = A.shape
    F = W_gu_interleaved.shape[0] // 2
    require(W_gu_interleaved.shape[1] == K and tuple(act.shape) == (M, F), "swiglu shapes")
    check(load_library().yapd_gemm_swiglu(A.data_ptr(), A.stride(0), W_gu_interleaved.data_ptr(), M, F, K,
                                          act.data_ptr(), act.stride(0), stream_ptr(dev)))


def interleave_gate_up(w_gate: torch.Tensor, w_up: torch.Tensor) -> torch.Tensor:
    """Rows ``[g(32w..32w+31); u(32w..32w+31)]`` for w = 0..F/32-1: gate and up of a
    feature land in the same lane of the swiglu epilogue."""
    F, K = w_gate.shape
    require(F % 64 == 0 and w_up.shape == w_gate.shape, "gate/up must be [F, K] with F % 64 == 0")
    return torch.stack([w_gate.view(F // 32, 32, K), w_up.view(F // 32, 32, K)], 1).reshape(2 * F, K).contiguous()


def gemm_qkv_rope_kv(A: torch.Tensor, W_qkv: torch.Tensor, cos_t: torch.Tensor, sin_t: torch.Tensor,
                     pos0: torch.Tensor, bl: int, q_out: torch.Tensor, pool: torch.Tensor,
                     table: torch.Tensor) -> None:
    """Fused QKV projection + NeoX RoPE + paged KV write (q to ``q_out [M, H*64]``).

    ``cos_t``/``sin_t`` are HF's [P, 64] tables (cat(freqs, freqs): column
    d + 32 equals column d); the kernel reads columns 0..31."""
    dev = A.device
    _mat(A, "A", dev)
    require_cuda(W_qkv, "W_qkv", torch.bfloat16, dev)
    M, K = A.shape
    H = pool.shape[2]
    require(tuple(W_qkv.shape) == (3 * H * 64, K), "W_qkv must be [3*H*64, K]")
    require_cuda(cos_t, "cos_t", torch.float32, dev)
    require_cuda(sin_t, "sin_t", torch.float32, dev)
    require(cos_t.shape == sin_t.shape and cos_t.dim() == 2 and cos_t.shape[1] == 64, "cos/sin must be [P, 64]")
    require_cuda(pos0, "pos0", torch.int32, dev)
    require(M % bl == 0 and pos0.numel() == M // bl, "pos0 must have M / bl entries")
    require_cuda(q_out, "q_out", torch.bfloat16, dev)
    require(tuple(q_out.shape) in ((M, H * 64), (M // bl, bl, H, 64)), "q_out shape")
    require_cuda(pool, "pool", torch.bfloat16, dev)
    require_cuda(table, "table", torch.int32, dev, contiguous=False)
    require(table.stride(1) == 1 and table.shape[0] >= M // bl, "table shape")
    check(load_library().yapd_gemm_qkv_rope_kv(
        A.data_ptr(), A.stride(0), W_qkv.data_ptr(), M, K, H, cos_t.data_ptr(), sin_t.data_ptr(), cos_t.shape[0],
        pos0.data_ptr(), bl, q_out.data_ptr(), pool.data_ptr(), pool.shape[0], table.data_ptr(), table.stride(0),
        table.shape[1], stream_ptr(dev)))


def gemm_rmsnorm_qkv_rope_kv(x: torch.Tensor, ln_w: torch.Tensor, eps: float, normed: torch.Tensor,
                             W_qkv: torch.Tensor, cos_t: torch.Tensor, sin_t: torch.Tensor, pos0: torch.Tensor,
                             bl: int, q_out: torch.Tensor, pool: torch.Tensor, table: torch.Tensor) -> None:
    """Input RMSNorm of the residual stream ``x [M, K]`` into ``normed`` (a caller workspace of the
    same shape), then :func:`gemm_qkv_rope_kv` on it (``yapd_gemm_rmsnorm_qkv_rope_kv``): two
    launches, not a fused kernel."""
    dev = x.device
    require_cuda(x, "x", torch.bfloat16, dev)
    require(x.dim() == 2, "x must be [M, K]")
    M, K = x.shape
    require_cuda(ln_w, "ln_w", torch.bfloat16, dev)
    require(ln_w.numel() == K, "ln_w must have K entries")
    require_cuda(normed, "normed", torch.bfloat16, dev)
    require(tuple(normed.shape) == (M, K), "normed must be [M, K]")
    require_cuda(W_qkv, "W_qkv", torch.bfloat16, dev)
    H = pool.shape[2]
    require(tuple(W_qkv.shape) == (3 * H * 64, K), "W_qkv must be [3*H*64, K]")
    require_cuda(cos_t, "cos_t", torch.float32, dev)
    require_cuda(sin_t, "sin_t", torch.float32, dev)
    require(cos_t.shape == sin_t.shape and cos_t.dim() == 2 and cos_t.shape[1] == 64, "cos/sin must be [P, 64]")
    require_cuda(pos0, "pos0", torch.int32, dev)
    require(M % bl == 0 and pos0.numel() == M // bl, "pos0 must have M / bl entries")
    require_cuda(q_out, "q_out", torch.bfloat16, dev)
    require(tuple(q_out.shape) in ((M, H * 64), (M // bl, bl, H, 64)), "q_out shape")
    require_cuda(pool, "pool", torch.bfloat16, dev)
    require_cuda(table, "table", torch.int32, dev, contiguous=False)
    require(table.stride(1) == 1 and table.shape[0] >= M // bl, "table shape")
    check(load_library().yapd_gemm_rmsnorm_qkv_rope_kv(
        x.data_ptr(), ln_w.data_ptr(), float(eps), normed.data_ptr(), W_qkv.data_ptr(), M, K, H, cos_t.data_ptr(),
        sin_t.data_ptr(), cos_t.shape[0], pos0.data_ptr(), bl, q_out.data_ptr(), pool.data_ptr(), pool.shape[0],
        table.data_ptr(), table.stride(0), table.shape[1], stream_ptr(dev)))


def rmsnorm(x: torch.Tensor, w: torch.Tensor, eps: float, out: torch.Tensor,
            delta: Optional[torch.Tensor] = None) -> None:
    """``out = rmsnorm(x) * w``; with ``delta``: ``x += delta`` (bf16, in place) first."""
    dev = x.device
    for name, t in (("x", x), ("w", w), ("out", out)):
        require_cuda(t, name, torch.bfloat16, dev)
    D = x.shape[-1]
    M = x.numel() // D
    require(out.shape == x.shape and w.numel() == D, "rmsnorm shapes")
    if delta is not None:
        require_cuda(delta, "delta", torch.bfloat16, dev)
        require(delta.shape == x.shape, "delta shape")
    check(load_library().yapd_rmsnorm(ptr(delta), x.data_ptr() if delta is not None else None,
                                      x.data_ptr() if delta is None else None, w.data_ptr(), float(eps), M, D,
                                      out.data_ptr(), stream_ptr(dev)))


def mfma_peak_probe(blocks: int, iters: int, out: torch.Tensor, random_operands: bool = True) -> float:
    """Launch the register-only MFMA calibration kernel (random or constant operands); returns its
    flop count."""
    require_cuda(out, "out", torch.float32, out.device)
    require(out.numel() >= blocks * 256, "out needs blocks * 256 floats")
    check(load_library().yapd_mfma_peak_probe(blocks, iters, int(bool(random_operands)), out.data_ptr(),
                                              stream_ptr(out.device)))
    return float(blocks) * 4 * iters * 8 * 32768


def hbm_read_probe(src: torch.Tensor, blocks: int, out: torch.Tensor) -> int:
    """Launch the streaming-read calibration kernel over all of ``src`` (contiguous, 16-byte aligned,
    a multiple of 16 bytes): workgroup b folds its contiguous share of 16-byte words, thread t of it the
    words b P + t, b P + t + 256, ... (P = the share rounded up to 256 words) by XOR into ``out[b * 256 + t]``.
    Returns the bytes read."""
    dev = src.device
    require(src.is_cuda and src.is_contiguous(), "src must be a contiguous GPU tensor")
    nbytes = src.numel() * src.element_size()
    require(nbytes % 16 == 0 and src.data_ptr() % 16 == 0, "src must be 16-byte aligned, a multiple of 16 bytes")
    require_cuda(out, "out", torch.int32, dev)
    require(out.numel() >= blocks * 256, "out needs blocks * 256 words")
    check(load_library().yapd_hbm_read_probe(src.data_ptr(), nbytes, blocks, out.data_ptr(), stream_ptr(dev)))
    return nbytes


def tick_update(*, xt: torch.Tensor, xt_blk: torch.Tensor, xt_new: torch.Tensor, k_step: torch.Tensor,
                cache_len: torch.Tensor, blk_start: torch.Tensor, is_commit: torch.Tensor, n_speech: torch.Tensor,
                hidden: torch.Tensor, shift_ctx: torch.Tensor, flags: torch.Tensor, xt_final: torch.Tensor,
                n_branch: int, K: int, mask_id: int, stop_id: int, max_len: int) -> None:
    """Continuous-batching state update after the scorer (``yapd_tick_update``) for the first
    ``xt_blk.shape[0]`` slots; every state tensor is updated in place."""
    dev = xt.device
    S, bl = xt_blk.shape
    D = hidden.shape[-1]
    for name, t in (("xt_blk", xt_blk), ("xt_new", xt_new), ("xt_final", xt_final)):
        require_cuda(t, name, torch.int64, dev)
        if not (tuple(t.shape) == (S, bl)):
            raise ValueError(f"{name} must be [slots, bl]")
    require_cuda(xt, "xt", torch.int64, dev, contiguous=False)
    require(xt.dim() == 2 and xt.stride(1) == 1 and xt.shape[0] >= S, "xt must be [slots, n_max] row-major")
    for name, t in (("k_step", k_step), ("cache_len", cache_len), ("blk_start", blk_start), ("n_speech", n_speech)):
        require_cuda(t, name, torch.int64, dev)
        if not (t.numel() >= S):
            raise ValueError(f"{name} needs one entry per slot")
    require_cuda(is_commit, "is_commit", torch.uint8, dev)
    require(is_commit.numel() >= S, "is_commit needs one entry per slot")
    require_cuda(hidden, "hidden", torch.bfloat16, dev)
    require(hidden.numel() >= S * n_branch * bl * D, "hidden must hold slots * n_branch * bl rows")
    require_cuda(shift_ctx, "shift_ctx", torch.bfloat16, dev)
    require(shift_ctx.numel() >= S * n_branch * D and shift_ctx.shape[-1] == D, "shift_ctx must be [rows, 1, D]")
    require_cuda(flags, "flags", torch.int64, dev)
    require(tuple(flags.shape) == (S, 6), "flags must be [slots, 6]")
    check(load_library().yapd_tick_update(
        S, bl, n_branch, D, K, mask_id, stop_id, max_len, xt.shape[1], xt.data_ptr(), xt.stride(0),
        xt_blk.data_ptr(), xt_new.data_ptr(), k_step.data_ptr(), cache_len.data_ptr(), blk_start.data_ptr(),
        is_commit.data_ptr(), n_speech.data_ptr(), hidden.data_ptr(), shift_ctx.data_ptr(), flags.data_ptr(),
        xt_final.data_ptr(), stream_ptr(dev)))


# --------------------------------------------------------------------------- #
# streaming vocoder: chunk stitching
# --------------------------------------------------------------------------- #

def voc_stitch(wav: torch.Tensor, jobs: torch.Tensor, fade_in: torch.Tensor, fade_out: torch.Tensor,
               trim: torch.Tensor, tails_in: Optional[torch.Tensor], tails_out: Optional[torch.Tensor],
               pcm: torch.Tensor) -> None:
    """Stitch a micro-batch's chunks into int16 PCM (``yapd_voc_stitch``, include/yapd_vocoder.h).

    ``wav`` fp32 ``[rows, S]`` with a unit last stride; ``jobs`` int32
    ``[n_jobs, 12]`` on the device (the layout of the header); ``fade_in`` /
    ``fade_out`` fp32 ``[fade]``; ``trim`` fp32 ``[n_trim]``; ``tails_in`` /
    ``tails_out`` fp32 ``[n, fade]`` or None; ``pcm`` int16, flat.
    """
    lib = load_library()
    dev = wav.device
    require_cuda(wav, "wav", torch.float32, dev, contiguous=False)
    require(wav.dim() == 2 and wav.stride(1) == 1, "wav must be [rows, samples] with unit last stride")
    require_cuda(jobs, "jobs", torch.int32, dev)
    if not (jobs.dim() == 2 and jobs.shape[1] == STITCH_JOB_INTS):
        raise ValueError(f"jobs must be [n, {STITCH_JOB_INTS}]")
    fade = fade_in.numel()
    for t, name in ((fade_in, "fade_in"), (fade_out, "fade_out"), (trim, "trim")):
        require_cuda(t, name, torch.float32, dev)
    require(fade_out.numel() == fade, "fade_in and fade_out must have the same length")
    for t, name in ((tails_in, "tails_in"), (tails_out, "tails_out")):
        if t is not None:
            require_cuda(t, name, torch.float32, dev)
            if not (t.dim() == 2 and t.shape[1] == fade):
                raise ValueError(f"{name} must be [n, {fade}]")
    require_cuda(pcm, "pcm", torch.int16, dev)
    n_in = 0 if tails_in is None else tails_in.shape[0]
    n_out = 0 if tails_out is None else tails_out.shape[0]
    check(lib.yapd_voc_stitch(wav.data_ptr(), wav.stride(0), wav.shape[1], wav.shape[0], jobs.data_ptr(),
                              jobs.shape[0], fade_in.data_ptr(), fade_out.data_ptr(), fade, ptr(trim),
                              trim.numel(), ptr(tails_in), n_in, ptr(tails_out), n_out, pcm.data_ptr(), pcm.numel(),
                              stream_ptr(dev)))
