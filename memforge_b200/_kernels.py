"""
Tensor-level wrappers over the C ABI.

PyTorch supplies device memory, streams and strides; every computation happens
in ``libmemforge_sm100.so``.  Tensors must be CUDA tensors: there is no CPU
implementation, and a CPU tensor is an error, not a reason to fall back.

Workspace and error word
------------------------
* The attention kernels keep split-K partials and arrival counters in a
  zero-initialised workspace they leave zeroed.  One is cached per device and
  grown on demand; make one warm-up call before capturing a CUDA graph so the
  capture does not allocate.  A workspace that is outgrown stays allocated, so
  graphs captured on it keep a valid address.  Launches on different streams
  that may overlap must pass their own ``workspace=``.
* Kernels report bad block ids, slots past the pool, too-short block tables and
  expired waits by OR-ing bits into a per-device int32 error word.  With
  ``MEMFORGE_CHECK=1`` (or ``set_checks(True)``) every call synchronises and
  raises on a non-zero word; otherwise ``check_device_errors()`` reads it.
"""

from __future__ import annotations

import ctypes
import os
import threading
from contextlib import nullcontext
from typing import Dict, Optional, Sequence, Tuple

import torch

from . import _lib as L

DTYPES = {torch.float32: L.MF_F32, torch.float16: L.MF_F16, torch.bfloat16: L.MF_BF16}

_state_lock = threading.Lock()
_workspaces: Dict[int, torch.Tensor] = {}
_retired: list = []   # grown-out workspaces, kept alive for graphs that captured them
_err_words: Dict[int, torch.Tensor] = {}
_checks = os.environ.get("MEMFORGE_CHECK", "0") not in ("", "0")
launch_counter = {"reshape_and_cache": 0, "paged_attention": 0, "copy_blocks": 0,
                  "peer_barrier": 0, "commit_window": 0, "gather_kv": 0,
                  "accept_commit": 0, "scored_attention": 0, "q4_reshape_and_cache": 0,
                  "q4_gather_kv": 0, "q4_paged_attention": 0}


def set_checks(enabled: bool) -> None:
    """Synchronise and check the device error word after every call."""
    global _checks
    _checks = bool(enabled)


def require_cuda(what: str, *tensors) -> None:
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise RuntimeError(
                f"{what}: memforge_b200 runs on CUDA tensors (sm_100a); got a tensor on {t.device}")


def dtype_code(dt: torch.dtype) -> int:
    if dt not in DTYPES:
        raise TypeError(f"unsupported dtype {dt}; expected float32, float16 or bfloat16")
    return DTYPES[dt]


def _dev_index(t: torch.Tensor) -> int:
    return t.device.index if t.device.index is not None else torch.cuda.current_device()


def err_word(device: torch.device) -> torch.Tensor:
    idx = device.index if device.index is not None else torch.cuda.current_device()
    w = _err_words.get(idx)
    if w is None:
        with _state_lock:
            w = _err_words.get(idx)
            if w is None:
                w = torch.zeros(1, dtype=torch.int32, device=torch.device("cuda", idx))
                _err_words[idx] = w
    return w


def check_device_errors(device: Optional[torch.device] = None, reset: bool = True) -> None:
    """Synchronise and raise if any kernel on `device` reported a violation."""
    device = device or torch.device("cuda", torch.cuda.current_device())
    w = err_word(device)
    bits = int(w.item())
    if reset and bits:
        w.zero_()
        idx = device.index if device.index is not None else torch.cuda.current_device()
        left = [ws for key, ws in list(_stream_workspaces.items()) if key[0] == idx]
        if left:
            torch.cuda.synchronize(device)   # other streams' launches may be using theirs
        if idx in _workspaces:
            left.append(_workspaces[idx])
        for ws in left:
            ws.zero_()   # an aborted launch may leave arrival counters behind
        if len(left) > 1:
            torch.cuda.synchronize(device)
    if bits:
        raise IndexError(f"memforge_b200 kernel reported: {L.describe_err(bits)} (0x{bits:x})")


def workspace(device: torch.device, nbytes: int) -> torch.Tensor:
    idx = device.index if device.index is not None else torch.cuda.current_device()
    ws = _workspaces.get(idx)
    if ws is None or ws.numel() < nbytes:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError(
                "paged attention needs a larger workspace during CUDA graph capture: make one "
                "call with the same shapes before capturing")
        with _state_lock:
            ws = _workspaces.get(idx)
            if ws is None or ws.numel() < nbytes:
                size = max(nbytes, 1 << 20)
                if ws is not None:
                    _retired.append(ws)
                ws = torch.zeros(size, dtype=torch.uint8, device=torch.device("cuda", idx))
                _workspaces[idx] = ws
    return ws


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream_ptr(device: torch.device) -> int:
    if _raw_stream is not None and device.index is not None:
        return _raw_stream(device.index)   # a tenth of current_stream()'s host time
    return torch.cuda.current_stream(device).cuda_stream


_err_ptrs: Dict[int, int] = {}


def _err_ptr(device: torch.device) -> int:
    p = _err_ptrs.get(device.index)
    if p is None:
        p = _err_ptrs[device.index] = err_word(device).data_ptr()
    return p


def _after(what: str, device: torch.device) -> None:
    if _checks:
        torch.cuda.synchronize(device)
        check_device_errors(device)


def _on(device: torch.device):
    """The tensors' device as the current one for a launch."""
    if device.index == torch.cuda.current_device():
        return nullcontext()
    return torch.cuda.device(device)


def require_one_device(what: str, device: torch.device, *tensors) -> None:
    for t in tensors:
        if t is None or (t.is_cuda and t.device == device):
            continue
        require_cuda(what, t)
        if t.device != device:
            raise ValueError(f"{what}: tensors on {device} and {t.device}")


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


# ------------------------------------------------------------------ KV write

def reshape_and_cache(key: torch.Tensor, value: torch.Tensor, key_pool: torch.Tensor,
                      value_pool: torch.Tensor, slot_mapping: torch.Tensor,
                      heads_major: bool = False) -> None:
    """
    Scatter ``key``/``value`` rows ``(T, H, D)`` (any strides, D contiguous)
    into one pool layer at ``slot_mapping[t]`` (int32/int64 CUDA tensor,
    -1 = skip).  ``key_pool`` is ``(blocks, block_size, H, D)``, or
    ``(blocks, H, block_size, D)`` with ``heads_major=True``.
    """
    require_cuda("reshape_and_cache", key, value, key_pool, value_pool, slot_mapping)
    if key.dim() != 3 or value.shape != key.shape:
        raise ValueError(f"keys/values must be (T, H, D) of one shape, got {tuple(key.shape)} "
                         f"and {tuple(value.shape)}")
    if key.stride(-1) != 1:
        key = key.contiguous()
    if value.stride(-1) != 1:
        value = value.contiguous()
    if key_pool.stride(-1) != 1 or value_pool.stride() != key_pool.stride():
        raise ValueError("pool layers must share strides and have a contiguous last dim")
    if slot_mapping.dtype not in (torch.int32, torch.int64):
        raise TypeError("slot_mapping must be int32 or int64")
    if not slot_mapping.is_contiguous():
        slot_mapping = slot_mapping.contiguous()
    T, H, D = key.shape
    if heads_major:
        nb, hp, bs, dp = key_pool.shape
        sb, sh, ss = key_pool.stride(0), key_pool.stride(1), key_pool.stride(2)
    else:
        nb, bs, hp, dp = key_pool.shape
        sb, ss, sh = key_pool.stride(0), key_pool.stride(1), key_pool.stride(2)
    if (hp, dp) != (H, D):
        raise ValueError(f"pool holds {hp} heads x {dp} dims, keys are {H} x {D}")
    if slot_mapping.numel() != T:
        raise ValueError(f"{T} tokens but {slot_mapping.numel()} slots")
    if T == 0:
        return
    lib = L.lib()
    dev = key.device
    rc = lib.mf_reshape_and_cache(
        key.data_ptr(), value.data_ptr(), dtype_code(key.dtype), key.stride(0), key.stride(1),
        value.stride(0), value.stride(1), key_pool.data_ptr(), value_pool.data_ptr(),
        dtype_code(key_pool.dtype), sb, ss, sh, nb, bs, slot_mapping.data_ptr(),
        1 if slot_mapping.dtype == torch.int64 else 0, T, H, D, err_word(dev).data_ptr(),
        _stream_ptr(dev))
    L.check(rc, "mf_reshape_and_cache")
    launch_counter["reshape_and_cache"] += 1
    _after("reshape_and_cache", dev)


def gather_kv(key_pool: torch.Tensor, value_pool: torch.Tensor, flat_index: torch.Tensor,
              heads_major: bool = False):
    """
    ``mf_gather_kv``: the pool slots ``flat_index`` (int32/int64 CUDA tensor) of
    one layer ``(blocks, block_size, H, D)`` (or ``(blocks, H, block_size, D)``
    with ``heads_major``) as contiguous ``(1, H, T, D)`` keys and values.
    """
    require_cuda("gather_kv", key_pool, value_pool)
    if flat_index.device != key_pool.device:
        flat_index = flat_index.to(key_pool.device)
    if key_pool.stride(-1) != 1 or value_pool.stride() != key_pool.stride():
        raise ValueError("pool layers must share strides and have a contiguous last dim")
    if flat_index.dtype not in (torch.int32, torch.int64):
        raise TypeError("flat_index must be int32 or int64")
    flat_index = flat_index.reshape(-1).contiguous()
    if heads_major:
        nb, H, bs, D = key_pool.shape
        sb, sh, ss = key_pool.stride(0), key_pool.stride(1), key_pool.stride(2)
    else:
        nb, bs, H, D = key_pool.shape
        sb, ss, sh = key_pool.stride(0), key_pool.stride(1), key_pool.stride(2)
    T = flat_index.numel()
    k = torch.empty((1, H, T, D), dtype=key_pool.dtype, device=key_pool.device)
    v = torch.empty_like(k)
    if T == 0:
        return k, v
    dev = key_pool.device
    rc = L.lib().mf_gather_kv(key_pool.data_ptr(), value_pool.data_ptr(),
                              dtype_code(key_pool.dtype), sb, ss, sh, nb, bs,
                              flat_index.data_ptr(), 1 if flat_index.dtype == torch.int64 else 0,
                              T, H, D, k.data_ptr(), v.data_ptr(), T * D, D,
                              err_word(dev).data_ptr(), _stream_ptr(dev))
    L.check(rc, "mf_gather_kv")
    launch_counter["gather_kv"] += 1
    _after("gather_kv", dev)
    return k, v


def commit_window(win_k: torch.Tensor, win_v: torch.Tensor, key_pool: torch.Tensor,
                  value_pool: torch.Tensor, block_tables: torch.Tensor, ctx_lens: torch.Tensor,
                  num_confirmed: torch.Tensor) -> None:
    """
    Write rows ``0 .. num_confirmed[b]-1`` of each sequence's window into the
    pool at positions ``ctx_lens[b] + j`` (one launch; the slot arithmetic runs
    on the device).  One layer: ``win_k``/``win_v`` ``(B*W, H, D)``
    sequence-major and ``key_pool`` ``(blocks, block_size, H, D)``; every layer
    at once: ``(L, B*W, H, D)`` windows and ``(L, blocks, block_size, H, D)``
    pools.  ``block_tables`` int32 ``[B, width]``, ``ctx_lens`` and
    ``num_confirmed`` int32 ``[B]``.  Rows past ``num_confirmed`` are not
    written.
    """
    require_cuda("commit_window", win_k, win_v, key_pool, value_pool, block_tables, ctx_lens,
                 num_confirmed)
    if win_v.shape != win_k.shape or win_k.dim() not in (3, 4):
        raise ValueError(f"window keys/values must be (B*W, H, D) or (L, B*W, H, D) of one "
                         f"shape, got {tuple(win_k.shape)} and {tuple(win_v.shape)}")
    layered = win_k.dim() == 4
    if key_pool.dim() != (5 if layered else 4) or value_pool.shape != key_pool.shape:
        raise ValueError("pools must be (blocks, block_size, H, D) for (B*W, H, D) windows and "
                         "(L, blocks, block_size, H, D) for (L, B*W, H, D) windows")
    wk = win_k if layered else win_k.unsqueeze(0)
    wv = win_v if layered else win_v.unsqueeze(0)
    kp = key_pool if layered else key_pool.unsqueeze(0)
    vp = value_pool if layered else value_pool.unsqueeze(0)
    B = ctx_lens.numel()
    if B == 0:
        return
    if num_confirmed.numel() != B:
        raise ValueError(f"{B} sequences but {num_confirmed.numel()} confirmed counts")
    L_, R, H, D = wk.shape
    W = R // B
    if W * B != R or W == 0:
        raise ValueError("window rows are not a whole number of windows")
    if kp.shape[0] != L_:
        raise ValueError(f"{L_} window layers but {kp.shape[0]} pool layers")
    if wk.stride(-1) != 1:
        wk = wk.contiguous()
    if wv.stride(-1) != 1:
        wv = wv.contiguous()
    if kp.stride(-1) != 1 or vp.stride() != kp.stride():
        raise ValueError("pools must share strides and have a contiguous last dim")
    _, nb, bs, hp, dp = kp.shape
    if (hp, dp) != (H, D):
        raise ValueError(f"pool holds {hp} heads x {dp} dims, window rows are {H} x {D}")
    if block_tables.dim() != 2 or block_tables.shape[0] != B:
        raise ValueError("block_tables must be [B, width]")
    tables = block_tables.to(torch.int32).contiguous()
    ctx = ctx_lens.to(torch.int32).contiguous()
    conf = num_confirmed.to(torch.int32).contiguous()
    dev = win_k.device
    rc = L.lib().mf_commit_window(
        wk.data_ptr(), wv.data_ptr(), dtype_code(wk.dtype), wk.stride(0), wk.stride(1),
        wk.stride(2), wv.stride(0), wv.stride(1), wv.stride(2), kp.data_ptr(), vp.data_ptr(),
        dtype_code(kp.dtype), kp.stride(0), kp.stride(1), kp.stride(2), kp.stride(3), L_, nb, bs,
        tables.data_ptr(), tables.stride(0), ctx.data_ptr(), conf.data_ptr(), B, W, H, D,
        err_word(dev).data_ptr(), _stream_ptr(dev))
    L.check(rc, "mf_commit_window")
    launch_counter["commit_window"] += 1
    _after("commit_window", dev)


def copy_blocks(key_pool: torch.Tensor, value_pool: torch.Tensor, pairs: torch.Tensor) -> None:
    """Copy block src -> dst in every layer; ``pairs`` is int32 ``[n, 2]`` on the device."""
    require_cuda("copy_blocks", key_pool, value_pool, pairs)
    if not (key_pool.is_contiguous() and value_pool.is_contiguous()):
        raise ValueError("copy_blocks needs contiguous pools")
    if pairs.dtype != torch.int32:
        pairs = pairs.to(torch.int32)
    pairs = pairs.contiguous()
    layers, nb = key_pool.shape[0], key_pool.shape[1]
    block_elems = key_pool[0, 0].numel()
    dev = key_pool.device
    rc = L.lib().mf_copy_blocks(key_pool.data_ptr(), value_pool.data_ptr(), layers, nb,
                                block_elems, key_pool.element_size(), pairs.data_ptr(),
                                pairs.shape[0], err_word(dev).data_ptr(), _stream_ptr(dev))
    L.check(rc, "mf_copy_blocks")
    launch_counter["copy_blocks"] += 1
    _after("copy_blocks", dev)


# ----------------------------------------------------------------- attention

def paged_attention(q: torch.Tensor, out: torch.Tensor, key_pool: torch.Tensor,
                    value_pool: torch.Tensor, block_tables: torch.Tensor,
                    kv_lens: torch.Tensor, *, cu_seqlens_q: Optional[torch.Tensor] = None,
                    q_per_seq: int = 1, max_q_len: Optional[int] = None, scale: float,
                    causal: bool = True, row_map: Optional[torch.Tensor] = None,
                    win_k: Optional[torch.Tensor] = None, win_v: Optional[torch.Tensor] = None,
                    heads_major: bool = False, workspace_tensor: Optional[torch.Tensor] = None,
                    out_peers: Optional[Sequence[int]] = None, out_head_offset: int = 0,
                    softcap: float = 0.0, window: int = 0,
                    alibi_slopes: Optional[torch.Tensor] = None,
                    prefix_lens: Optional[torch.Tensor] = None) -> torch.Tensor:
    """
    ``mf_paged_attention`` on torch tensors.

    q, out: ``(rows, Hq, D)`` views (any row/head strides, D contiguous).
    key_pool/value_pool: one layer, ``(blocks, block_size, Hkv, D)`` (or
    ``(blocks, Hkv, block_size, D)`` with ``heads_major``).
    block_tables: int32 ``[num_seqs, width]``; kv_lens: int32 ``[num_seqs]``;
    cu_seqlens_q: int32 ``[num_seqs+1]`` or None (uniform ``q_per_seq``);
    row_map: int32 ``[rows]`` or None; win_k/win_v: ``(rows, Hkv, D)`` or None.
    out_peers: device addresses of the full ``[rows, total heads, D]`` output on
    every GPU of a head-sharded step (``out`` gives their strides); the kernel
    stores this call's heads at ``out_head_offset`` into all of them.
    softcap / window / alibi_slopes / prefix_lens: the score modifiers of
    ``mf_paged_attention_scored`` (0 or None: none; slopes fp32 ``[Hq]``, prefixes int32
    ``[num_seqs]``).  Without ``workspace_tensor`` a call with modifiers uses a
    workspace of its device and stream, and inside a graph capture one of its own.
    """
    require_cuda("paged_attention", q, out, key_pool, value_pool, block_tables, kv_lens,
                 cu_seqlens_q, row_map, win_k, win_v)
    for name, t in (("block_tables", block_tables), ("kv_lens", kv_lens),
                    ("cu_seqlens_q", cu_seqlens_q), ("row_map", row_map)):
        if t is not None and t.dtype != torch.int32:
            raise TypeError(f"{name} must be int32 (got {t.dtype})")
    if q.stride(-1) != 1 or out.stride(-1) != 1:
        raise ValueError("q/out need a contiguous head_dim")
    if key_pool.stride() != value_pool.stride() or key_pool.stride(-1) != 1:
        raise ValueError("pool layers must share strides and have a contiguous last dim")
    if q.dtype != key_pool.dtype or out.dtype != q.dtype or value_pool.dtype != q.dtype:
        raise TypeError("q, out and the pool must share a dtype")
    if block_tables.dim() != 2 or block_tables.stride(1) != 1:
        block_tables = block_tables.contiguous()
    kv_lens = kv_lens.contiguous()
    rows, hq, d = q.shape
    if heads_major:
        nb, hkv, bs, dp = key_pool.shape
        sb, sh, ss = key_pool.stride(0), key_pool.stride(1), key_pool.stride(2)
    else:
        nb, bs, hkv, dp = key_pool.shape
        sb, ss, sh = key_pool.stride(0), key_pool.stride(1), key_pool.stride(2)
    if dp != d:
        raise ValueError(f"query head_dim {d} but the pool holds {dp}")
    num_seqs = kv_lens.numel()
    a = L.AttentionArgs()
    a.struct_size = ctypes_sizeof_args()
    a.q, a.q_stride_row, a.q_stride_head = q.data_ptr(), q.stride(0), q.stride(1)
    a.out, a.out_stride_row, a.out_stride_head = out.data_ptr(), out.stride(0), out.stride(1)
    a.k_pool, a.v_pool = key_pool.data_ptr(), value_pool.data_ptr()
    a.pool_stride_block, a.pool_stride_slot, a.pool_stride_head = sb, ss, sh
    a.num_blocks, a.block_size = nb, bs
    a.block_tables, a.table_stride = block_tables.data_ptr(), block_tables.stride(0)
    a.cu_seqlens_q = _ptr(cu_seqlens_q)
    a.q_per_seq = q_per_seq
    a.kv_lens = kv_lens.data_ptr()
    a.row_map = _ptr(row_map)
    if win_k is not None:
        if win_k.stride() != win_v.stride() or win_k.stride(-1) != 1:
            raise ValueError("window K/V must share strides with a contiguous last dim")
        a.win_k, a.win_v = win_k.data_ptr(), win_v.data_ptr()
        a.win_stride_row, a.win_stride_head = win_k.stride(0), win_k.stride(1)
    a.num_seqs, a.total_q = num_seqs, rows
    a.max_q_len = max_q_len if max_q_len is not None else q_per_seq
    a.num_q_heads, a.num_kv_heads, a.head_dim = hq, hkv, d
    a.scale, a.causal, a.dtype = float(scale), 1 if causal else 0, dtype_code(q.dtype)
    if out_peers:
        if len(out_peers) > L.MF_MAX_OUT_PEERS:
            raise ValueError(f"at most {L.MF_MAX_OUT_PEERS} output peers")
        a.num_out_peers, a.out_head_offset = len(out_peers), int(out_head_offset)
        for i, ptr in enumerate(out_peers):
            a.out_peers[i] = int(ptr)
    lib = L.lib()
    dev = q.device
    idx = _dev_index(q)
    mods = score_mods(dev, hq, num_seqs, softcap, window, alibi_slopes, prefix_lens)
    if mods is not None:
        require_one_device("paged_attention", dev, out, key_pool, value_pool, block_tables,
                           kv_lens, cu_seqlens_q, row_map, workspace_tensor)
        if out.shape != q.shape or value_pool.shape != key_pool.shape:
            raise ValueError(f"out must have q's shape and the value pool the key pool's, got "
                             f"{tuple(out.shape)} for {tuple(q.shape)} and "
                             f"{tuple(value_pool.shape)} for {tuple(key_pool.shape)}")
        if block_tables.dim() != 2 or block_tables.shape[0] < num_seqs:
            raise ValueError("block_tables must be [num_seqs, width]")
        if cu_seqlens_q is not None and (cu_seqlens_q.numel() != num_seqs + 1 or max_q_len is None
                                         or not cu_seqlens_q.is_contiguous()):
            raise ValueError("cu_seqlens_q needs num_seqs + 1 contiguous offsets and max_q_len")
        if row_map is not None and (row_map.numel() < rows or not row_map.is_contiguous()):
            raise ValueError("row_map must be contiguous with an entry for each row")
        with _on(dev):
            need = lib.mf_paged_attention_scored_workspace_size(a, mods, idx)
            ws = workspace_tensor if workspace_tensor is not None else (
                stream_workspace(dev, need) if need else None)
            rc = lib.mf_paged_attention_scored(a, mods, _ptr(ws), 0 if ws is None else ws.numel(),
                                               err_word(dev).data_ptr(), _stream_ptr(dev))
        L.check(rc, "mf_paged_attention_scored")
        launch_counter["scored_attention"] += 1
        _after("scored_attention", dev)
        return out
    need = lib.mf_paged_attention_workspace_size(a, idx)
    ws = workspace_tensor if workspace_tensor is not None else (
        workspace(dev, need) if need else None)
    rc = lib.mf_paged_attention(a, _ptr(ws), 0 if ws is None else ws.numel(),
                                err_word(dev).data_ptr(), _stream_ptr(dev))
    L.check(rc, "mf_paged_attention")
    launch_counter["paged_attention"] += 1
    _after("paged_attention", dev)
    return out


def score_mods(device: torch.device, num_q_heads: int, num_seqs: int, softcap: float, window: int,
               alibi_slopes: Optional[torch.Tensor],
               prefix_lens: Optional[torch.Tensor]) -> Optional[L.ScoreMods]:
    """The checked ``mf_score_mods``, or None when no modifier is given."""
    if not softcap and not window and alibi_slopes is None and prefix_lens is None:
        return None
    if softcap != 0.0 and not 1e-30 <= softcap <= 1e30:
        raise ValueError(f"softcap must be 0 (none) or from 1e-30 to 1e30, got {softcap}")
    if window < 0:
        raise ValueError(f"window must be 0 (none) or positive, got {window}")
    for name, t, dt, n in (("alibi_slopes", alibi_slopes, torch.float32, num_q_heads),
                           ("prefix_lens", prefix_lens, torch.int32, num_seqs)):
        if t is None:
            continue
        if t.device != device or t.dtype != dt or t.numel() != n or not t.is_contiguous():
            raise ValueError(f"{name} must be {n} contiguous {dt} values on {device}, got "
                             f"{tuple(t.shape)} {t.dtype} on {t.device}")
    # (int32 on the other side; a wider window hides nothing either)
    return L.ScoreMods(float(softcap), min(int(window), 2 ** 31 - 1), _ptr(alibi_slopes), _ptr(prefix_lens))


_stream_workspaces: Dict[Tuple[int, int], torch.Tensor] = {}


def stream_workspace(device: torch.device, nbytes: int) -> torch.Tensor:
    """
    A zeroed-counter workspace that no other stream uses: one per (device, stream), or,
    inside a graph capture, memory of that graph whose counters the graph clears.
    """
    if torch.cuda.is_current_stream_capturing():
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
        ws[:min(nbytes, 1 << 20)].zero_()   # the arrival counters at its front
        return ws
    key = (device.index, _stream_ptr(device))
    ws = _stream_workspaces.get(key)
    if ws is None or ws.numel() < nbytes:
        ws = torch.zeros(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
        _stream_workspaces[key] = ws
    return ws


# ------------------------------------------------------------- 4-bit KV cache

Q4_BLOCK = 16


def q4_head_dim(pool: torch.Tensor) -> int:
    """head_dim of a 4-bit pool layer ``(blocks, kv_heads, 16 * D + 128)``, checked."""
    return _q4_layer(pool, None)[5]


def _q4_layer(pool: torch.Tensor, layer: Optional[int]):
    """(address, block stride, head stride, blocks, kv heads, head_dim) of one layer of a
    4-bit pool ``([layers,] blocks, kv_heads, 16 * D + 128)``, without a view of it."""
    shape, stride = pool.shape, pool.stride()
    want = 3 if layer is None else 4
    if pool.dtype != torch.uint8 or len(shape) != want or stride[-1] != 1:
        raise ValueError(f"a 4-bit pool is uint8 ({'' if layer is None else 'layers, '}blocks, "
                         f"kv_heads, 16 * D + 128) with contiguous records, got {pool.dtype} "
                         f"{tuple(shape)}")
    d = (shape[-1] - 128) // 16
    if d not in (64, 128, 256) or shape[-1] != 16 * d + 128:
        raise ValueError(f"no head_dim of 64, 128 or 256 has records of {shape[-1]} bytes")
    ptr = pool.data_ptr()
    if layer is not None:
        if not -shape[0] <= layer < shape[0]:
            raise IndexError(f"layer {layer} of a pool of {shape[0]}")
        ptr += (layer % shape[0]) * stride[0]
    return ptr, stride[-3], stride[-2], shape[-3], shape[-2], d


def _slots(name: str, t: torch.Tensor) -> torch.Tensor:
    if t.dtype != torch.int64 and t.dtype != torch.int32:
        raise TypeError(f"{name} must be int32 or int64")
    return t if t.is_contiguous() else t.contiguous()


def q4_reshape_and_cache(key: torch.Tensor, value: torch.Tensor, pool: torch.Tensor,
                         slot_mapping: torch.Tensor, *, layer: Optional[int] = None,
                         heads_first: bool = False) -> None:
    """
    ``mf_q4_reshape_and_cache``: quantise ``key``/``value`` rows ``(T, H, D)`` (fp32,
    fp16 or bf16, any token and head strides) into one 4-bit pool layer
    ``(blocks, H, 16 * D + 128)`` at ``slot_mapping[t]`` (-1 = skip).  ``layer``: that
    layer of a pool ``(layers, blocks, H, 16 * D + 128)``.  ``heads_first``: rows come as
    ``(1, H, T, D)``.
    """
    dev = pool.device
    require_one_device("q4_reshape_and_cache", dev, pool, key, value, slot_mapping)
    ptr, sb, sh, nb, ph, D = _q4_layer(pool, layer)
    shape = key.shape
    if value.shape != shape or value.dtype != key.dtype or len(shape) != (4 if heads_first else 3):
        raise ValueError(f"keys/values must be {'(1, H, T, D)' if heads_first else '(T, H, D)'} of "
                         f"one shape and dtype, got {tuple(shape)} {key.dtype} and "
                         f"{tuple(value.shape)} {value.dtype}")
    ks, vs = key.stride(), value.stride()
    if ks[-1] != 1:
        key = key.contiguous()
        ks = key.stride()
    if vs[-1] != 1:
        value = value.contiguous()
        vs = value.stride()
    if heads_first:
        one, H, T, d = shape
        if one != 1:
            raise ValueError(f"keys/values must be (1, heads, tokens, head_dim), got "
                             f"{tuple(shape)}")
        kst, ksh, vst, vsh = ks[2], ks[1], vs[2], vs[1]
    else:
        T, H, d = shape
        kst, ksh, vst, vsh = ks[0], ks[1], vs[0], vs[1]
    if (H, d) != (ph, D):
        raise ValueError(f"pool holds {ph} heads x {D} dims, keys are {H} x {d}")
    slots = _slots("slot_mapping", slot_mapping)
    if slots.numel() != T:
        raise ValueError(f"{T} tokens but {slots.numel()} slots")
    code = dtype_code(key.dtype)
    if T == 0:
        return
    args = (key.data_ptr(), value.data_ptr(), code, kst, ksh, vst, vsh, ptr, sb, sh, nb,
            slots.data_ptr(), 1 if slots.dtype == torch.int64 else 0, T, H, D, _err_ptr(dev),
            _stream_ptr(dev))
    if dev.index == torch.cuda.current_device():
        rc = L.lib().mf_q4_reshape_and_cache(*args)
    else:
        with torch.cuda.device(dev):
            rc = L.lib().mf_q4_reshape_and_cache(*args)
    if rc:
        L.check(rc, "mf_q4_reshape_and_cache")
    launch_counter["q4_reshape_and_cache"] += 1
    if _checks:
        _after("q4_reshape_and_cache", dev)


def q4_gather_kv(pool: torch.Tensor, flat_index: torch.Tensor, dtype: torch.dtype, *,
                 layer: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """
    ``mf_q4_gather_kv``: slots ``flat_index`` of one 4-bit pool layer, dequantised to
    contiguous ``(1, H, T, D)`` keys and values of ``dtype``.
    """
    dev = pool.device
    require_cuda("q4_gather_kv", pool)
    ptr, sb, sh, nb, H, D = _q4_layer(pool, layer)
    code = dtype_code(dtype)
    if flat_index.device != dev:
        flat_index = flat_index.to(dev)
    index = _slots("flat_index", flat_index)
    T = index.numel()
    k = torch.empty((1, H, T, D), dtype=dtype, device=dev)
    v = torch.empty_like(k)
    if T == 0:
        return k, v
    args = (ptr, sb, sh, nb, index.data_ptr(), 1 if index.dtype == torch.int64 else 0, T, H, D,
            k.data_ptr(), v.data_ptr(), code, T * D, D, _err_ptr(dev), _stream_ptr(dev))
    if dev.index == torch.cuda.current_device():
        rc = L.lib().mf_q4_gather_kv(*args)
    else:
        with torch.cuda.device(dev):
            rc = L.lib().mf_q4_gather_kv(*args)
    if rc:
        L.check(rc, "mf_q4_gather_kv")
    launch_counter["q4_gather_kv"] += 1
    if _checks:
        _after("q4_gather_kv", dev)
    return k, v


_q4_need: Dict[tuple, int] = {}   # workspace bytes by the sizes they depend on


def q4_paged_attention(q: torch.Tensor, out: torch.Tensor, pool: torch.Tensor,
                       block_tables: torch.Tensor, kv_lens: torch.Tensor, *,
                       cu_seqlens_q: Optional[torch.Tensor] = None, q_per_seq: int = 1,
                       max_q_len: Optional[int] = None, scale: float, causal: bool = True,
                       row_map: Optional[torch.Tensor] = None, softcap: float = 0.0,
                       window: int = 0, alibi_slopes: Optional[torch.Tensor] = None,
                       prefix_lens: Optional[torch.Tensor] = None,
                       workspace_tensor: Optional[torch.Tensor] = None,
                       layer: Optional[int] = None) -> torch.Tensor:
    """
    ``mf_q4_paged_attention`` on torch tensors: q, out ``(rows, Hq, D)`` views (any row
    and head strides, D contiguous), one 4-bit pool layer (``layer``: of a pool with a
    layer dimension), and tables, lengths, rows and score modifiers as in
    :func:`paged_attention`.  The workspace is scratch of the caching allocator unless
    one is given; where it has no room for the expanded copy that long runs read, they
    convert the cache as they go.
    """
    dev = q.device
    require_one_device("q4_paged_attention", dev, q, out, pool, block_tables, kv_lens,
                       cu_seqlens_q, row_map, workspace_tensor)
    ptr, sb, sh, nb, hkv, D = _q4_layer(pool, layer)
    i32 = torch.int32
    if block_tables.dtype != i32 or kv_lens.dtype != i32 or (
            cu_seqlens_q is not None and cu_seqlens_q.dtype != i32) or (
            row_map is not None and row_map.dtype != i32):
        raise TypeError("block_tables, kv_lens, cu_seqlens_q and row_map must be int32")
    shape, qs, os_ = q.shape, q.stride(), out.stride()
    if len(shape) != 3 or out.shape != shape or out.dtype != q.dtype:
        raise ValueError(f"q and out must be (rows, heads, D) of one shape and dtype, got "
                         f"{tuple(shape)} {q.dtype} and {tuple(out.shape)} {out.dtype}")
    if qs[2] != 1 or os_[2] != 1:
        raise ValueError("q/out need a contiguous head_dim")
    rows, hq, d = shape
    if d != D:
        raise ValueError(f"query head_dim {d} but the pool holds {D}")
    if hq % hkv:
        raise ValueError(f"{hq} query heads is not a multiple of {hkv} kv heads")
    num_seqs = kv_lens.numel()
    if block_tables.dim() != 2 or block_tables.shape[0] != num_seqs:
        raise ValueError("block_tables must be [num_seqs, width]")
    if cu_seqlens_q is not None:
        if cu_seqlens_q.numel() != num_seqs + 1 or max_q_len is None:
            raise ValueError("cu_seqlens_q needs num_seqs + 1 offsets and max_q_len")
        if not cu_seqlens_q.is_contiguous():
            cu_seqlens_q = cu_seqlens_q.contiguous()
        most = int(max_q_len)
    else:
        if q_per_seq * num_seqs != rows:
            raise ValueError(f"{num_seqs} sequences of {q_per_seq} rows but {rows} query rows")
        most = q_per_seq
    if row_map is not None and (row_map.numel() < rows or not row_map.is_contiguous()):
        raise ValueError("row_map must be contiguous with an entry for each row")
    ts = block_tables.stride()
    if ts[1] != 1:
        block_tables = block_tables.contiguous()
        ts = block_tables.stride()
    if not kv_lens.is_contiguous():
        kv_lens = kv_lens.contiguous()
    width, code = block_tables.shape[1], dtype_code(q.dtype)
    if rows == 0:
        return out
    a = L.Q4AttentionArgs(
        ctypes.sizeof(L.Q4AttentionArgs), q.data_ptr(), qs[0], qs[1], out.data_ptr(), os_[0],
        os_[1], ptr, sb, sh, nb, block_tables.data_ptr(), ts[0], width, _ptr(cu_seqlens_q),
        q_per_seq, kv_lens.data_ptr(), _ptr(row_map), num_seqs, rows, most, hq, hkv, D, scale,
        1 if causal else 0, code)
    mods = score_mods(dev, hq, num_seqs, softcap, window, alibi_slopes, prefix_lens)
    if mods is not None:
        a.mods = mods
    lib = L.lib()
    ws, nbytes, fresh = workspace_tensor, 0, False
    if ws is None:
        key = (dev.index, code, D, hq, hkv, num_seqs, most, width, cu_seqlens_q is None,
               mods is None, rows, (a.q | a.out | 2 * (qs[0] | qs[1] | os_[0] | os_[1])) & 15)
        nbytes = _q4_need.get(key)
        fresh = nbytes is None
        if fresh:
            nbytes = lib.mf_q4_paged_attention_workspace_size(a, dev.index)
        if nbytes:
            try:
                ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
            except torch.OutOfMemoryError:
                least = lib.mf_q4_paged_attention_min_workspace_size(a, dev.index)
                if least >= nbytes:
                    raise
                # no room for the expanded copy (and it is not kept as the size of such calls)
                nbytes, fresh = least, False
                ws = torch.empty(least, dtype=torch.uint8, device=dev) if least else None
    else:
        nbytes = ws.numel() * ws.element_size()
    args = (a, _ptr(ws), nbytes, _err_ptr(dev), _stream_ptr(dev))
    if dev.index == torch.cuda.current_device():
        rc = lib.mf_q4_paged_attention(*args)
    else:
        with torch.cuda.device(dev):
            rc = lib.mf_q4_paged_attention(*args)
    if rc:
        L.check(rc, "mf_q4_paged_attention")
    if fresh:   # (not of a refused call, whose size of 0 says nothing)
        if len(_q4_need) > 4096:
            _q4_need.clear()
        _q4_need[key] = nbytes
    launch_counter["q4_paged_attention"] += 1
    if _checks:
        _after("q4_paged_attention", dev)
    return out


_ARGS_SIZE = None


def ctypes_sizeof_args() -> int:
    global _ARGS_SIZE
    if _ARGS_SIZE is None:
        _ARGS_SIZE = ctypes.sizeof(L.AttentionArgs)
    return _ARGS_SIZE


def peer_barrier(flag_ptrs: Sequence[int], rank: int, epoch: int,
                 device: torch.device) -> None:
    """``mf_peer_barrier``: completes a head-sharded step (see ``kv_shard.PeerOutput``)."""
    arr = (ctypes.c_void_p * len(flag_ptrs))(*[int(p) for p in flag_ptrs])
    rc = L.lib().mf_peer_barrier(arr, len(flag_ptrs), int(rank), int(epoch),
                                 err_word(device).data_ptr(), _stream_ptr(device))
    L.check(rc, "mf_peer_barrier")
    launch_counter["peer_barrier"] += 1
