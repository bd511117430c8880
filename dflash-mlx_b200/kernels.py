"""GatedDeltaNet tape recording and tape replay on B200.

Mirrors ``dflash_mlx/kernels.py``:

* ``gated_delta_kernel_with_tape(q, k, v, g, beta, state, mask=None)`` --
  ``kernels.py:169-219``: the verify forward over T steps returning
  ``(y, state, tape)`` (y bf16 ``[B, T, Hv, Dv]``, new fp32 state, fp32
  innovation tape); q, k, v bf16, g and beta fp32.  Its state updates are the
  replay's operations in the same order, so replaying its tape over a prefix
  of a steps gives exactly its state after a steps.
* ``tape_replay_kernel(tape, k, g, state, mask=None)`` -- ``kernels.py:822-868``.
  Functional like the reference: returns a new state and leaves ``state``
  untouched.  Same shapes: tape fp32 ``[B, T, Hv, Dv]``, k ``[B, T, Hk, Dk]``
  (bf16 or fp32), g ``[B, T, Hv]`` or ``[B, T, Hv, Dk]``, state fp32
  ``[B, Hv, Dv, Dk]``, optional bool mask ``[B, T]``.
* ``tape_replay_(state, tape, k, g, steps, mask)`` -- the in-place form the
  rollback uses on B200: replays the first ``steps[b]`` steps of each
  sequence and does not touch sequences with nothing to replay.
* ``gated_delta_rule(q, k, v, g, beta, state, ...)`` -- the same recurrence
  without a tape, for prompts of any length (padded with a mask, or packed
  with ``cu_seqlens``) and for single tokens; the reference runs it through
  mlx-lm's ``gated_delta_update`` for caches that are not armed
  (``engine/target_qwen_gdn.py:551-651``).

The update per replayed step is ``S <- S * g_t`` then ``S <- S + delta_t k_t``,
two separately rounded fp32 operations in the order of the mx-op reference
(``kernels.py:790-820``).  Only fp32 states are supported (the reference
re-rounds the state to its own dtype after every step, ``kernels.py:745-747``,
which is the identity for fp32).
"""

from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _lib
from ._runtime import mask_bytes, on_device, overlap, require_cuda, same_device, stream_ptr


def _check(tape, k, g, state, steps=None, mask=None):
    for t, name in ((tape, "tape"), (k, "k"), (g, "g"), (state, "state")):
        require_cuda(t, name)
    if state.dtype != torch.float32:
        raise NotImplementedError(f"state must be float32, got {state.dtype}")
    if tape.dtype != torch.float32:
        raise NotImplementedError(f"tape must be float32, got {tape.dtype}")
    if k.dtype not in (torch.bfloat16, torch.float32):
        raise NotImplementedError(f"k must be bfloat16 or float32, got {k.dtype}")
    if g.dtype != torch.float32:
        raise NotImplementedError(f"g must be float32, got {g.dtype}")
    b, t_steps, hk, dk = k.shape
    hv, dv = tape.shape[2:]
    if hv % hk != 0:
        raise ValueError(f"Cannot align K heads {hk} to tape heads {hv}")
    if tape.shape[:2] != (b, t_steps):
        raise ValueError("tape and k disagree on [B, T]")
    if state.shape != (b, hv, dv, dk):
        raise ValueError(f"state must be [B, Hv, Dv, Dk] = {(b, hv, dv, dk)}, got {tuple(state.shape)}")
    if g.dim() == 3:
        if g.shape != (b, t_steps, hv):
            raise ValueError("scalar g must be [B, T, Hv]")
    elif g.dim() == 4:
        if g.shape != (b, t_steps, hv, dk):
            raise ValueError("vector g must be [B, T, Hv, Dk]")
    else:
        raise ValueError(f"Unsupported gating shape {tuple(g.shape)}")
    # the kernel reads steps[b] for every sequence and mask[b, t] for every step
    if steps is not None and steps.numel() != b:
        raise ValueError(f"steps must hold one count per sequence ({b}), got {steps.numel()}")
    if mask is not None and mask.numel() != b * t_steps:
        raise ValueError(f"mask must be [B, T] = {(b, t_steps)}, got {tuple(mask.shape)}")
    return b, t_steps, hv, hk, dv, dk


def _launch(tape, k, g, state_in, state_out, steps, mask, dims):
    b, t_steps, hv, hk, dv, dk = dims
    tape = tape.contiguous()
    k = k.contiguous()
    g = g.contiguous()
    steps_ptr = 0
    mask_ptr = 0
    if steps is not None:
        steps = steps.to(device=state_in.device, dtype=torch.int32).contiguous()
        steps_ptr = steps.data_ptr()
    if mask is not None:
        mask = mask.to(device=state_in.device, dtype=torch.uint8).contiguous()
        mask_ptr = mask.data_ptr()
    with torch.cuda.device(state_in.device):
        st = _lib.load().dfl_gdn_tape_replay(
            tape.data_ptr(), k.data_ptr(), 1 if k.dtype == torch.bfloat16 else 0, g.data_ptr(),
            1 if g.dim() == 4 else 0, steps_ptr or None, mask_ptr or None, state_in.data_ptr(),
            state_out.data_ptr(), b, t_steps, hv, hk, dv, dk, stream_ptr(state_in.device))
    _lib.check("dfl_gdn_tape_replay", st)
    return state_out


def tape_replay_kernel(tape: torch.Tensor, k: torch.Tensor, g: torch.Tensor, state: torch.Tensor,
                       mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Replay the recorded innovation tape onto ``state`` (reference ``kernels.py:822``)."""
    dims = _check(tape, k, g, state, mask=mask)
    state = state.contiguous()
    out = torch.empty_like(state)
    return _launch(tape, k, g, state, out, None, mask, dims)


def tape_replay_(state: torch.Tensor, tape: torch.Tensor, k: torch.Tensor, g: torch.Tensor,
                 steps: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """In-place replay of the first ``steps[b]`` steps of each sequence, without
    those whose ``mask [B, T]`` is False."""
    if not state.is_contiguous():
        raise ValueError("in-place replay needs a contiguous state")
    dims = _check(tape, k, g, state, steps=steps, mask=mask)
    return _launch(tape, k, g, state, state, steps, mask, dims)


def gated_delta_kernel_with_tape(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor,
                                 beta: torch.Tensor, state: torch.Tensor,
                                 mask: Optional[torch.Tensor] = None):
    """GDN verify forward recording the innovation tape (reference ``kernels.py:169``).

    Returns ``(y, new_state, tape)``; ``state`` is left untouched.
    """
    for t, name in ((q, "q"), (k, "k"), (v, "v"), (g, "g"), (beta, "beta"), (state, "state")):
        require_cuda(t, name)
    for t, name in ((q, "q"), (k, "k"), (v, "v")):
        if t.dtype != torch.bfloat16:
            raise NotImplementedError(f"{name} must be bfloat16, got {t.dtype}")
    if g.dtype != torch.float32 or beta.dtype != torch.float32:
        raise NotImplementedError("g and beta must be float32")
    if state.dtype != torch.float32:
        raise NotImplementedError(f"state must be float32, got {state.dtype}")
    b, t_steps, hk, dk = k.shape
    hv, dv = v.shape[2:]
    if q.shape != k.shape:
        raise ValueError("q and k must have the same shape")
    if hv % hk != 0:
        raise ValueError(f"Cannot align K heads {hk} to V heads {hv}")
    if v.shape[:2] != (b, t_steps) or beta.shape != (b, t_steps, hv):
        raise ValueError("v must be [B, T, Hv, Dv] and beta [B, T, Hv]")
    if g.shape not in ((b, t_steps, hv), (b, t_steps, hv, dk)):
        raise ValueError(f"Unsupported gating shape {tuple(g.shape)}")
    if state.shape != (b, hv, dv, dk):
        raise ValueError(f"state must be [B, Hv, Dv, Dk] = {(b, hv, dv, dk)}, got {tuple(state.shape)}")
    q, k, v, g, beta, state = (t.contiguous() for t in (q, k, v, g, beta, state))
    y = torch.empty((b, t_steps, hv, dv), dtype=torch.bfloat16, device=state.device)
    tape = torch.empty((b, t_steps, hv, dv), dtype=torch.float32, device=state.device)
    out = torch.empty_like(state)
    mask_ptr = None
    if mask is not None:
        mask = mask.to(device=state.device, dtype=torch.uint8).reshape(b, t_steps).contiguous()
        mask_ptr = mask.data_ptr()
    with torch.cuda.device(state.device):
        st = _lib.load().dfl_gdn_forward_tape(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), 1 if g.dim() == 4 else 0,
            beta.data_ptr(), mask_ptr, state.data_ptr(), out.data_ptr(), y.data_ptr(),
            tape.data_ptr(), b, t_steps, hv, hk, dv, dk, stream_ptr(state.device))
    _lib.check("dfl_gdn_forward_tape", st)
    return y, out, tape


# ------------------------------------------------- whole sequences, no tape
def _token_rows(x: torch.Tensor, b: int, t: int, h: int, d: int):
    """``x [B, T, H, D]`` as tokens one fixed stride apart: ``(tensor, stride)``.
    Views of a wider projection (heads and values next to each other, tokens
    further apart) are read in place when their rows are 16-byte aligned;
    everything else is copied."""
    if x.data_ptr() % 16 == 0:
        if x.is_contiguous():
            return x, h * d
        s0, s1, s2, s3 = x.stride()
        step = s1 if t > 1 else (s0 if b > 1 else h * d)
        if (s3 == 1 and (h == 1 or s2 == d) and step >= h * d and (b == 1 or t == 1 or s0 == t * step)
                and step % 8 == 0 and step < 2**31):
            return x, step
    return _aligned(x), h * d


def gated_delta_rule(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor,
                     beta: torch.Tensor, state: torch.Tensor, *, mask: Optional[torch.Tensor] = None,
                     cu_seqlens: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                     out_state: Optional[torch.Tensor] = None):
    """The gated delta rule over whole sequences: ``(y, new_state)``.

    ``q, k [B, T, Hk, Dk]`` and ``v [B, T, Hv, Dv]`` bf16 (views of a wider
    projection output are read in place), ``g [B, T, Hv]`` or ``[B, T, Hv,
    Dk]`` and ``beta [B, T, Hv]`` fp32; ``y`` bf16 ``[B, T, Hv, Dv]``.

    * Padded batch: ``state`` fp32 ``[B, Hv, Dv, Dk]``, optional bool ``mask
      [B, T]``; a step whose mask is False leaves the state, its ``y`` is 0 and
      what its inputs hold does not matter.
    * Packed: ``B = 1`` and ``cu_seqlens`` int32 ``[N + 1]`` on the device;
      sequence n is tokens ``cu_seqlens[n] .. cu_seqlens[n + 1] - 1`` (lengths
      of 0 and 1 included) and starts from ``state[n]``, ``[N, Hv, Dv, Dk]``.

    ``out`` receives y (rows that belong to no sequence are left as they were;
    a new y has zeros there) and shares no memory with the inputs or
    ``out_state``.  ``out_state`` receives the new state and may be ``state``
    itself, whole or in part, but meets no other input; without it ``state`` is
    left untouched.  Nothing is read back to the host; the call can
    be captured into a CUDA graph.  A NaN or an infinity in a step that counts
    reaches what follows it, as in the recurrence, and may reach the y of up to
    63 steps before it where steps are taken 64 at a time (from a mean length of
    some 20 to 64 steps on, Dk 64 or 128, one decay per head).

    Keys are such that ``beta |k|^2 < 2``, as for any use of the rule (above that a
    step stretches the state, and what it errs grows with it).  States are then
    right to 32-bit sums in both forms, 1e-7 to 8e-7 of their 2-norm for keys of unit
    length at any angles; y to its rounding to bf16.

    Sequences of one call are taken one way, by their mean length.  So a long
    prompt and many single tokens belong in two calls: 4096 steps and 300 single
    tokens of 48 heads of 128 x 128 take 3.5 ms in one pack, 0.33 + 0.36 ms apart.
    """
    require_cuda(state, "state")
    dev = state.device
    same_device(dev, q=q, k=k, v=v, g=g, beta=beta, mask=mask, cu_seqlens=cu_seqlens, out=out,
                out_state=out_state)
    bf16, f32 = torch.bfloat16, torch.float32
    if q.dtype != bf16 or k.dtype != bf16 or v.dtype != bf16:
        raise NotImplementedError(f"q, k and v must be bfloat16, got {q.dtype}, {k.dtype}, {v.dtype}")
    if g.dtype != f32 or beta.dtype != f32 or state.dtype != f32:
        raise NotImplementedError(f"g, beta and state must be float32, got {g.dtype}, {beta.dtype}, {state.dtype}")
    if k.dim() != 4 or v.dim() != 4:
        raise ValueError(f"q, k and v must be [B, T, heads, dim], got {tuple(k.shape)} and {tuple(v.shape)}")
    b, t_steps, hk, dk = k.shape
    bv, tv, hv, dv = v.shape
    if q.shape != k.shape:
        raise ValueError("q and k must have the same shape")
    if hk < 1 or hv < 1 or hv % hk != 0:
        raise ValueError(f"Cannot align K heads {hk} to V heads {hv}")
    if dk not in (32, 64, 128, 256) or dv < 32 or dv % 32 != 0:
        raise ValueError(f"Dk must be 32, 64, 128 or 256 and Dv a multiple of 32, got {dk} and {dv}")
    tokens = (b, t_steps, hv)
    if bv != b or tv != t_steps or beta.shape != tokens:
        raise ValueError("v must be [B, T, Hv, Dv] and beta [B, T, Hv]")
    vector = g.dim() == 4
    if g.shape != ((b, t_steps, hv, dk) if vector else tokens):
        raise ValueError(f"Unsupported gating shape {tuple(g.shape)}")
    seqs, steps, cu_ptr, mask_ptr = b, t_steps, None, None
    if cu_seqlens is not None:
        if b != 1:
            raise ValueError(f"packed sequences take B = 1, got {b}")
        if cu_seqlens.dtype != torch.int32 or cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1:
            raise ValueError("cu_seqlens must be int32 [sequences + 1]")
        cu_seqlens = cu_seqlens.contiguous()
        cu_ptr = cu_seqlens.data_ptr()
        seqs = cu_seqlens.numel() - 1
        steps = t_steps // max(seqs, 1)
    shape = (seqs, hv, dv, dk)
    if state.shape != shape:
        raise ValueError(f"state must be [B, Hv, Dv, Dk] = {shape}, got {tuple(state.shape)}")
    if mask is not None:
        if mask.shape != (b, t_steps):
            raise ValueError(f"mask must be [B, T] = {(b, t_steps)}, got {tuple(mask.shape)}")
        mask = mask_bytes(mask, "mask")
        mask_ptr = mask.data_ptr()
    zero_gaps = out is None
    if out is None:
        new = torch.zeros if seqs == 0 else torch.empty
        out = new((b, t_steps, hv, dv), dtype=bf16, device=dev)
    elif (out.dtype != bf16 or out.shape != (b, t_steps, hv, dv) or not out.is_contiguous()
          or out.data_ptr() % 16 != 0):
        raise ValueError(f"out must be contiguous, 16-byte aligned bf16 {(b, t_steps, hv, dv)}")
    elif overlap(out, q, k, v, g, beta, mask, cu_seqlens, state, out_state):
        raise ValueError("out must not share memory with an input or out_state")
    if out_state is None:
        out_state = torch.empty(shape, dtype=f32, device=dev)
        state = _aligned(state)
    else:
        if (out_state.dtype != f32 or out_state.shape != shape or not out_state.is_contiguous()
                or out_state.data_ptr() % 16 != 0):
            raise ValueError(f"out_state must be contiguous, 16-byte aligned fp32 {shape}")
        if overlap(out_state, q, k, v, g, beta, mask, cu_seqlens):
            raise ValueError("out_state must not share memory with an input other than state")
        if out_state.data_ptr() == state.data_ptr() and state.is_contiguous():
            pass   # in place
        elif overlap(out_state, state):
            state = state.clone(memory_format=torch.contiguous_format)   # in part
        else:
            state = _aligned(state)
    q, ldq = _token_rows(q, b, t_steps, hk, dk)
    k, ldk = _token_rows(k, b, t_steps, hk, dk)
    v, ldv = _token_rows(v, b, t_steps, hv, dv)
    g, beta = g.contiguous(), beta.contiguous()
    lib = _lib.load()
    head = (q.data_ptr(), ldq, k.data_ptr(), ldk, v.data_ptr(), ldv, g.data_ptr())
    tail = (beta.data_ptr(), mask_ptr, cu_ptr, state.data_ptr(), out_state.data_ptr(), out.data_ptr(),
            1 if zero_gaps else 0, seqs, t_steps, hv, hk, dv, dk)
    with on_device(dev):
        if not vector and (dk == 128 or dk == 64) and steps >= _chunked_from(seqs * hv * -(-dv // 128), dv, dk):
            entry = "dfl_gdn_rule_chunked"
            status = ctypes.c_int(0)
            n = lib.dfl_gdn_rule_workspace_bytes(seqs, t_steps, 0 if cu_ptr is None else 1, hv, dv, dk,
                                                 ctypes.byref(status))
            _lib.check("dfl_gdn_rule_workspace_bytes", status.value)
            ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
            st = lib.dfl_gdn_rule_chunked(*head, *tail, ws.data_ptr() if n else None, n, stream_ptr(dev))
        else:
            entry = "dfl_gdn_rule_recurrent"
            st = lib.dfl_gdn_rule_recurrent(*head, 1 if vector else 0, *tail, stream_ptr(dev))
    if st:
        _lib.check(entry, st)
    return out, out_state


def _chunked_from(tiles: int, dv: int, dk: int) -> int:
    """Mean steps of a sequence from which 64 steps at a time are faster than
    one after the other.  A chunk takes much the same time for any size of the
    state (up to 128 rows) and has an SM to itself, so small states need more
    steps once there are more of them than SMs.  Measured, us one after the
    other and 64 at a time, 16, 24 and 64 steps: one sequence of 48 heads of 128 x
    128 13 / 15.6, 18.6 / 15.8 and 44 / 15.2, equal at 20, 40 of those 193 / 197, 273 /
    195 and 670 / 189; 80 heads of 64 x 64 9 / 13.2, 12.5 / 13.4 and 28 / 13.1; 320
    of those 13 / 35.5, 18 / 35 and 40 / 34.8; 320 heads of 128 x 64 (Dv x Dk) 19 / 42.6,
    26 / 42 and 62 / 41, equal at 40 steps.  Sequences of one call take one form
    together, whatever their own lengths (they are known on the device only)."""
    size = dk * min(dv, 128)
    if size >= 128 * 128:
        return 20
    if tiles <= 148:
        return 26
    return 40 if size >= 128 * 64 else 64


def _aligned(x: torch.Tensor) -> torch.Tensor:
    """``x`` contiguous with 16-byte aligned storage."""
    x = x.contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone()


# ------------------------------------------------------------------ DDTree
def _tree_inputs(q, k, v, g, beta, state, parent_ids):
    for t, name in ((q, "q"), (k, "k"), (v, "v"), (g, "g"), (beta, "beta"), (state, "state")):
        require_cuda(t, name)
    if q.dtype not in (torch.bfloat16, torch.float32) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise NotImplementedError("q, k, v must all be bfloat16 or all float32")
    if state.dtype != torch.float32:
        raise NotImplementedError(f"state must be float32, got {state.dtype}")
    b, t_steps, hk, dk = k.shape
    hv, dv = v.shape[2:]
    if q.shape != k.shape:
        raise ValueError("q and k must have the same shape")
    if hv % hk != 0:
        raise ValueError(f"Cannot align K heads {hk} to V heads {hv}")
    if g.shape not in ((b, t_steps, hv), (b, t_steps, hv, dk)):
        raise ValueError(f"Unsupported gating shape {tuple(g.shape)}")
    if beta.shape != (b, t_steps, hv) or state.shape != (b, hv, dv, dk):
        raise ValueError("beta must be [B, T, Hv] and state [B, Hv, Dv, Dk]")
    parent_ids = torch.as_tensor(parent_ids).to(device=state.device, dtype=torch.int32).reshape(-1)
    if parent_ids.numel() != t_steps:
        raise ValueError("parent_ids must have one entry per tree node")
    # g and beta enter the kernel as fp32 (bf16 values widen exactly)
    g = g.to(torch.float32)
    beta = beta.to(torch.float32)
    q, k, v, g, beta, state, parent_ids = (x.contiguous() for x in (q, k, v, g, beta, state, parent_ids))
    return q, k, v, g, beta, state, parent_ids, (b, t_steps, hv, hk, dv, dk)


def _tree_launch(q, k, v, g, beta, state, parent_ids, dims, want_tape):
    b, t_steps, hv, hk, dv, dk = dims
    y = torch.empty((b, t_steps, hv, dv), dtype=q.dtype, device=state.device)
    nodes = torch.empty((b, t_steps, hv, dv, dk), dtype=torch.float32, device=state.device)
    tape = torch.empty((b, t_steps, hv, dv), dtype=torch.float32, device=state.device) if want_tape else None
    with torch.cuda.device(state.device):
        st = _lib.load().dfl_gdn_tree_forward(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), 1 if g.dim() == 4 else 0,
            beta.data_ptr(), state.data_ptr(), parent_ids.data_ptr(), y.data_ptr(), nodes.data_ptr(),
            tape.data_ptr() if tape is not None else None, b, t_steps, hv, hk, dv, dk,
            1 if q.dtype == torch.float32 else 0, stream_ptr(state.device))
    _lib.check("dfl_gdn_tree_forward", st)
    return y, nodes, tape


def gated_delta_tree_kernel(q, k, v, g, beta, state, parent_ids):
    """GDN over a token tree (reference ``kernels.py:501``): ``(y, tree_states)``,
    node t starting from node ``parent_ids[t]`` (or ``state`` when < 0)."""
    q, k, v, g, beta, state, parent_ids, dims = _tree_inputs(q, k, v, g, beta, state, parent_ids)
    y, nodes, _ = _tree_launch(q, k, v, g, beta, state, parent_ids, dims, want_tape=False)
    return y, nodes


def gated_delta_tree_tape_kernel(q, k, v, g, beta, state, parent_ids):
    """The tree recurrence recording the innovation tape (reference
    ``kernels.py:545``): ``(y, tape)``; replaying a root-to-node path's tape rows
    with ``tape_replay_kernel`` reproduces that node's state."""
    q, k, v, g, beta, state, parent_ids, dims = _tree_inputs(q, k, v, g, beta, state, parent_ids)
    y, _, tape = _tree_launch(q, k, v, g, beta, state, parent_ids, dims, want_tape=True)
    return y, tape


def tree_depthwise_conv1d(qkv, prefix, weight, bias, path_indices):
    """Depthwise conv1d along tree paths + SiLU (reference ``kernels.py:647``).

    ``qkv [B, T, C]``, ``prefix [B, K-1, C]`` (same dtype, bf16 or fp32),
    ``weight [C, K, 1]`` (or ``[C, K]``), ``bias [C]`` or None,
    ``path_indices [T, K]`` into ``concat(prefix, qkv)``."""
    for t, name in ((qkv, "qkv"), (prefix, "prefix"), (weight, "weight")):
        require_cuda(t, name)
    if qkv.dtype not in (torch.bfloat16, torch.float32):
        raise NotImplementedError(f"qkv must be bfloat16 or float32, got {qkv.dtype}")
    b, t_steps, c = qkv.shape
    w = weight[..., 0] if weight.dim() == 3 else weight
    if w.shape[0] != c:
        raise ValueError(f"weight must be [C, K(, 1)] with C = {c}")
    kk = int(w.shape[1])
    if prefix.shape != (b, kk - 1, c) or prefix.dtype != qkv.dtype:
        raise ValueError(f"prefix must be [B, K-1, C] = {(b, kk - 1, c)} in qkv's dtype")
    if bias is not None and bias.numel() != c:
        raise ValueError(f"bias must hold one value per channel ({c}), got {bias.numel()}")
    path = torch.as_tensor(path_indices).to(device=qkv.device, dtype=torch.int32).reshape(t_steps, kk)
    w = w.to(torch.float32).contiguous()
    bias = bias.to(device=qkv.device, dtype=torch.float32).contiguous() if bias is not None else None
    qkv, prefix, path = qkv.contiguous(), prefix.contiguous(), path.contiguous()
    out = torch.empty_like(qkv)
    with torch.cuda.device(qkv.device):
        st = _lib.load().dfl_tree_depthwise_conv1d(
            qkv.data_ptr(), prefix.data_ptr(), w.data_ptr(), bias.data_ptr() if bias is not None else None,
            path.data_ptr(), out.data_ptr(), b, t_steps, c, kk, 1 if qkv.dtype == torch.float32 else 0,
            stream_ptr(qkv.device))
    _lib.check("dfl_tree_depthwise_conv1d", st)
    return out
