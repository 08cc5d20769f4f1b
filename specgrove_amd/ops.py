"""Torch-facing wrappers of the HIP kernels (PyTorch is only the memory and
stream plumbing here: tensors are passed to the C ABI as raw device pointers,
and every call is enqueued on torch's current HIP stream).

Argument checks follow the reference's native-op conventions
(fused_tree_sampling.py:158-174, :472-509): contiguity/device/dtype problems
raise ValueError before anything is launched; launch errors raise RuntimeError.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass, field, replace

import numpy as np
import torch

from . import _lib


# Raw handle of torch's current stream without building a Stream object
# (torch.cuda.current_stream() costs ~3 us per call, this ~0.1 us).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream_handle() -> int:
    """torch's current HIP stream on the current device."""
    if _raw_stream is not None:
        return _raw_stream(torch.cuda.current_device())
    return torch.cuda.current_stream().cuda_stream


class PreparedCall:
    """A validated C-ABI call whose argument struct is built once.

    Calling it only enqueues the kernels on torch's current stream, so a
    caller that repeats a call over the same buffers (a decode loop over
    persistent staging) pays the argument checks and the struct once.  It
    holds the tensors it points to: their contents may change between calls,
    their storage, shapes and strides may not.  Returns ``result``.
    """
    __slots__ = ("_fn", "_ref", "_args", "_keep", "_name", "result")

    def __init__(self, fn_name: str, args, keep, result=None):
        self._fn = getattr(_lib.load(), fn_name)
        self._args = args
        self._ref = ctypes.byref(args)
        self._keep = keep
        self._name = fn_name
        self.result = result

    def __call__(self):
        _lib.check(self._fn(self._ref, _stream_handle()), self._name)
        return self.result

    def set(self, **fields) -> "PreparedCall":
        """Update scalar fields of the bound argument struct (sizes and
        strides that change from call to call over the same buffers, e.g. a
        commit's request count); the library checks them on every call."""
        for name, value in fields.items():
            if not hasattr(self._args, name):
                raise ValueError(f"{self._name} has no argument {name}")
            setattr(self._args, name, value)
        return self


_upload_streams: dict = {}  # device index -> the stream of upload()'s copies


def upload(array: np.ndarray, device) -> torch.Tensor:
    """A host array on the device, complete on return: any stream, graph
    capture or thread may read it without waiting.  The copy runs on a stream
    of its own into memory of that stream, so the host waits for the copy (36
    to 39 us for 32 KiB; 24 us on the current stream while it is idle) and not
    for the current stream's earlier work.  (While a stream is captured the
    copy is a plain one, which capture refuses.)"""
    host = torch.from_numpy(array)
    device = torch.device(device)
    if device.type != "cuda" or torch.cuda.is_current_stream_capturing():
        return host.to(device)
    index = torch.cuda.current_device() if device.index is None else device.index
    stream = _upload_streams.get(index)
    if stream is None:
        stream = _upload_streams.setdefault(index, torch.cuda.Stream(index))
    with torch.cuda.stream(stream):
        copy = host.to(device)
    copy.record_stream(torch.cuda.current_stream(index))
    return copy


def _require(cond: bool, message: str) -> None:
    if not cond:
        raise ValueError(message)


def _check_device_tensor(t: torch.Tensor, name: str, dtype: torch.dtype) -> None:
    if isinstance(t, torch.Tensor) and t.is_cuda and t.dtype == dtype:
        return
    _require(isinstance(t, torch.Tensor), f"{name} must be a tensor")
    _require(t.is_cuda, f"{name} must be a HIP device tensor")
    _require(t.dtype == dtype, f"{name} must be {dtype}, got {t.dtype}")


def _check_device_tensors(tensors: tuple, names: tuple, dtype: torch.dtype) -> None:
    """_check_device_tensor over several tensors of one dtype."""
    for t in tensors:
        if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype == dtype):
            break
    else:
        return
    for t, name in zip(tensors, names):
        _check_device_tensor(t, name, dtype)


def _check_rows(t: torch.Tensor, name: str) -> None:
    """bf16 tensors whose last (head) dim is contiguous and 16-byte aligned."""
    _check_device_tensor(t, name, torch.bfloat16)
    st = t.stride()
    if st[-1] == 1 and t.data_ptr() % 16 == 0 and not any(s % 8 for s in st[:-1]):
        return
    _require(st[-1] == 1, f"{name} must have a contiguous last dimension")
    _require(t.data_ptr() % 16 == 0, f"{name} must be 16-byte aligned")
    _require(not any(s % 8 for s in st[:-1]), f"{name} strides must be multiples of 8 elements")


# --------------------------------------------------------------------------
# (A) attention
# --------------------------------------------------------------------------

@dataclass
class AttnPlan:
    """Host-built work list of the packed attention (one per wave, all layers)."""
    host: np.ndarray
    units: int
    merges: int
    workspace_bytes: int
    num_q_heads: int
    num_kv_heads: int
    head_dim: int
    device: torch.Tensor | None = None
    workspace: torch.Tensor | None = None
    # What the plan was made from, and the wave's plan over a 4-bit cache (in_mx4).
    wave: tuple | None = field(default=None, repr=False, compare=False)
    # (No copy by dataclasses.replace carries it: its memory is not the copy's.)
    mx4: "AttnPlan | None" = field(default=None, init=False, repr=False, compare=False)

    @property
    def header(self) -> np.ndarray:
        """The plan header as int32 words (see decode_plan)."""
        return self.host[:64].view(np.int32)

    @property
    def num_requests(self) -> int:
        return int(self.header[8])

    @property
    def num_rows(self) -> int:
        return int(self.header[9])

    def to(self, device) -> "AttnPlan":
        """Copy the plan to the device and allocate its workspace (the fp32
        partial results of split units; every slot is written before the merge
        kernel reads it, so its initial contents do not matter)."""
        self.device = torch.from_numpy(self.host).to(device, non_blocking=False)
        self.workspace = torch.zeros(max(self.workspace_bytes, 16), dtype=torch.uint8,
                                     device=device)
        self.mx4 = None  # of the device before
        return self

    def with_workspace(self) -> "AttnPlan":
        """The same plan on the device with a workspace of its own, of the
        current stream's memory: calls that can overlap, as on two streams,
        must not share one."""
        plan = replace(self, workspace=torch.empty(
            max(self.workspace_bytes, 16), dtype=torch.uint8, device=self.device.device))
        if self.mx4 is not None and self.mx4.device.device == self.device.device:
            plan.mx4 = self.mx4.with_workspace()
        return plan

    def in_mx4(self) -> "AttnPlan":
        """The plan that ``tree_attention_mx4`` runs of this one: itself if it was made
        for a 4-bit cache or a given number of units, else ``plan_attention_mx4`` of the
        same wave, made and copied at the first use on a device and kept (not while a
        stream is captured: use the plan once before).  Its workspace is memory of the
        stream of that first use; another stream takes a ``with_workspace()`` of the plan."""
        if self.wave is None:
            return self
        if self.mx4 is None or self.mx4.device.device != self.device.device:
            check_plan(self, *self.wave)  # the host copy may have been replaced
            _require(not torch.cuda.is_current_stream_capturing(),
                     "the plan's 4-bit form is made at its first use: call once before a "
                     "capture, or use plan_attention_mx4")
            plan = plan_attention_mx4(*self.wave, self.num_q_heads, self.num_kv_heads,
                                      self.head_dim)
            plan.device = upload(plan.host, self.device.device)
            self.mx4 = plan.with_workspace()
        return self.mx4


_PLAN_BYTES = 1 << 16  # about 1,300 units


def plan_attention(row_offset, prefix_len, num_q_heads: int, num_kv_heads: int,
                   head_dim: int, target_units: int = 0) -> AttnPlan:
    return _make_plan("sg_tree_attn_plan", row_offset, prefix_len, num_q_heads, num_kv_heads,
                      head_dim, target_units)


def plan_attention_mx4(row_offset, prefix_len, num_q_heads: int, num_kv_heads: int,
                       head_dim: int) -> AttnPlan:
    """``plan_attention`` for ``tree_attention_mx4``: prefixes cut for what the units
    take over a 4-bit cache."""
    return _make_plan("sg_tree_attn_plan_mx4", row_offset, prefix_len, num_q_heads,
                      num_kv_heads, head_dim)


def _make_plan(entry: str, row_offset, prefix_len, num_q_heads: int, num_kv_heads: int,
               head_dim: int, *hint: int) -> AttnPlan:
    make = getattr(_lib.load(), entry)
    ro = np.ascontiguousarray(np.asarray(row_offset, dtype=np.int32))
    pl = np.ascontiguousarray(np.asarray(prefix_len, dtype=np.int32))
    n = int(pl.size)
    _require(ro.size == n + 1, "row_offset must have num_requests + 1 entries")
    i32p = ctypes.POINTER(ctypes.c_int32)
    plan_bytes = ctypes.c_size_t()
    units = ctypes.c_int32()
    merges = ctypes.c_int32()
    ws = ctypes.c_size_t()
    args = (n, ro.ctypes.data_as(i32p), pl.ctypes.data_as(i32p), num_q_heads,
            num_kv_heads, head_dim, *hint)
    # The plan is made once, into a buffer that holds most plans; the size it
    # reports serves a larger one.
    host = np.empty(_PLAN_BYTES, dtype=np.uint8)
    for _ in range(2):
        rc = make(*args, host.ctypes.data_as(ctypes.c_void_p), host.nbytes,
                  ctypes.byref(plan_bytes), ctypes.byref(units), ctypes.byref(merges),
                  ctypes.byref(ws))
        if rc == 0 or plan_bytes.value <= host.nbytes:
            break
        host = np.empty(plan_bytes.value, dtype=np.uint8)
    _lib.check(rc, entry)
    host = host[:plan_bytes.value].copy()
    plan = AttnPlan(host, units.value, merges.value, ws.value, num_q_heads,
                    num_kv_heads, head_dim)
    if hint and hint[0] <= 0:  # cut by the planner's own rule: another cache, another cut
        plan.wave = (ro.copy(), pl.copy())
    return plan


def check_plan(plan: AttnPlan, row_offset_host, prefix_len_host) -> None:
    """Raise ValueError unless ``plan`` was built from exactly these row
    offsets and prefix lengths (plans are per wave: prefix lengths change
    after every commit)."""
    ro = np.ascontiguousarray(np.asarray(row_offset_host, dtype=np.int32))
    pl = np.ascontiguousarray(np.asarray(prefix_len_host, dtype=np.int32))
    _require(ro.size == pl.size + 1, "row_offset must have num_requests + 1 entries")
    i32p = ctypes.POINTER(ctypes.c_int32)
    _lib.check(_lib.load().sg_tree_attn_plan_check(
        plan.host.ctypes.data_as(ctypes.c_void_p), int(pl.size), ro.ctypes.data_as(i32p),
        pl.ctypes.data_as(i32p)), "sg_tree_attn_plan_check")


def check_plan_call(plan: AttnPlan, num_requests: int, num_rows: int, num_q_heads: int,
                    num_kv_heads: int, head_dim: int) -> None:
    """Host-side agreement of a plan with the call's shapes (no device access)."""
    _require((plan.num_q_heads, plan.num_kv_heads, plan.head_dim)
             == (num_q_heads, num_kv_heads, head_dim),
             "plan was built for another head configuration")
    header = plan.header
    requests, packed = int(header[8]), int(header[9])
    if requests != num_requests or packed != num_rows:
        raise ValueError(f"plan was built for another wave ({requests} requests, {packed} rows; "
                         f"the call has {num_requests} and {num_rows})")


UNIT_FIELDS = ("req", "kv_head", "row_begin", "row_count", "key_begin", "key_end",
               "partial", "flags", "group", "num_splits", "first_partial", "pad")


MERGE_FIELDS = ("req", "kv_head", "row_begin", "row_count", "first_partial", "num_partials",
                "pad0", "pad1")


def decode_plan(plan: AttnPlan):
    """(header [16], units [U, 12], merges [M, 8], bin_offset [B+1]) int32 views
    of a host plan; unit columns are UNIT_FIELDS, merge-group columns
    MERGE_FIELDS.  Work list b (workgroup b of the attention kernel) runs
    units[bin_offset[b]:bin_offset[b+1]]."""
    words = plan.host.view(np.int32)
    header = words[:16]
    n_units, n_merges, n_bins = int(header[1]), int(header[2]), int(header[7])
    end = 16 + len(UNIT_FIELDS) * n_units
    units = words[16:end].reshape(n_units, len(UNIT_FIELDS))
    mend = end + len(MERGE_FIELDS) * n_merges
    merges = words[end:mend].reshape(n_merges, len(MERGE_FIELDS))
    bins = words[mend:mend + n_bins + 1]
    return header, units, merges, bins


def tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                   k_tree: torch.Tensor, v_tree: torch.Tensor,
                   row_offset: torch.Tensor, prefix_start: torch.Tensor,
                   prefix_len: torch.Tensor, parent: torch.Tensor, plan: AttnPlan,
                   out: torch.Tensor | None = None, scale: float | None = None,
                   status: torch.Tensor | None = None) -> torch.Tensor:
    """Packed tree attention of one layer (see prepare_tree_attention)."""
    return prepare_tree_attention(q, k_cache, v_cache, k_tree, v_tree, row_offset,
                                  prefix_start, prefix_len, parent, plan, out=out,
                                  scale=scale, status=status)()


def prepare_tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                           k_tree: torch.Tensor, v_tree: torch.Tensor,
                           row_offset: torch.Tensor, prefix_start: torch.Tensor,
                           prefix_len: torch.Tensor, parent: torch.Tensor, plan: AttnPlan,
                           out: torch.Tensor | None = None, scale: float | None = None,
                           status: torch.Tensor | None = None) -> PreparedCall:
    """Packed tree attention of one layer, validated and bound (call it to run).

    q [R, Hq, D], k/v_cache [Hkv, tokens, D] (the cache arena of this layer),
    k/v_tree [R, Hkv, D] (this wave's rows), row_offset [n+1] i32,
    prefix_start [n] i64, prefix_len [n] i32, parent [R] i32.  Returns
    out [R, Hq, D] bf16.  ``status`` (optional [1] i32 device word, never
    cleared here) is set to SG_EINVAL by any unit whose key range or rows
    disagree with prefix_len / row_offset (a plan of another wave), whose
    output rows are then NaN.
    """
    for t, name in ((q, "q"), (k_cache, "k_cache"), (v_cache, "v_cache"),
                    (k_tree, "k_tree"), (v_tree, "v_tree")):
        _check_rows(t, name)
    _check_device_tensors((row_offset, prefix_len, parent),
                          ("row_offset", "prefix_len", "parent"), torch.int32)
    _check_device_tensor(prefix_start, "prefix_start", torch.int64)
    _require(q.dim() == 3 and k_tree.dim() == 3 and k_cache.dim() == 3,
             "q/k_tree must be [R, H, D] and k_cache [Hkv, tokens, D]")
    rows, hq, dim = q.shape
    hkv = k_cache.shape[0]
    cache_strides = k_cache.stride()
    tree_strides = k_tree.stride()
    _require(k_cache.shape == v_cache.shape and cache_strides == v_cache.stride(),
             "k_cache and v_cache must share shape and strides")
    _require(k_tree.shape == (rows, hkv, dim) and v_tree.shape == k_tree.shape
             and tree_strides == v_tree.stride(),
             "k_tree/v_tree must be [R, Hkv, D] with equal strides")
    _require(k_cache.shape[2] == dim, "head dims disagree")
    n = prefix_len.numel()
    check_plan_call(plan, n, rows, hq, hkv, dim)
    _require(plan.device is not None and plan.device.is_cuda, "plan is not on the device")
    _require(parent.numel() >= rows, "parent must cover every packed row")
    _require(row_offset.numel() == n + 1 and prefix_start.numel() == n,
             "request metadata sizes disagree")
    if status is not None:
        _check_device_tensor(status, "status", torch.int32)
    if out is None:
        out = torch.empty((rows, hq, dim), dtype=torch.bfloat16, device=q.device)
    _check_rows(out, "out")
    _require(out.shape == (rows, hq, dim), "out must be [R, Hq, D]")
    q_strides = q.stride()
    out_strides = out.stride()
    workspace = plan.workspace
    # Positional, in the order of SgTreeAttnArgs' fields.
    a = _lib.SgTreeAttnArgs(
        n, rows, hq, hkv, dim, float(dim ** -0.5 if scale is None else scale),
        q.data_ptr(), q_strides[0], q_strides[1],
        k_cache.data_ptr(), v_cache.data_ptr(), cache_strides[0], cache_strides[1],
        k_tree.data_ptr(), v_tree.data_ptr(), tree_strides[0], tree_strides[1],
        row_offset.data_ptr(), prefix_start.data_ptr(), prefix_len.data_ptr(),
        parent.data_ptr(), out.data_ptr(), out_strides[0], out_strides[1],
        plan.device.data_ptr(), plan.host.ctypes.data, plan.units, plan.merges,
        workspace.data_ptr() if workspace is not None else 0,
        workspace.numel() if workspace is not None else 0,
        status.data_ptr() if status is not None else 0)
    # The plan's tensors too: the plan may be moved and then holds others.
    keep = (q, k_cache, v_cache, k_tree, v_tree, row_offset, prefix_start, prefix_len, parent,
            plan.device, plan.host, workspace, out, status)
    return PreparedCall("sg_tree_attn_fwd", a, keep, result=out)


# --------------------------------------------------------------------------
# (B) KV commit
# --------------------------------------------------------------------------

def pointer_array(tensors, device) -> torch.Tensor:
    """Device array of the tensors' base addresses (int64)."""
    return torch.tensor([t.data_ptr() for t in tensors], dtype=torch.int64, device=device)


def kv_commit(k_cache_ptrs: torch.Tensor, v_cache_ptrs: torch.Tensor,
              k_tree_ptrs: torch.Tensor, v_tree_ptrs: torch.Tensor, **kw) -> None:
    """Scatter the kept rows of every layer into the cache (one call; see
    prepare_kv_commit)."""
    prepare_kv_commit(k_cache_ptrs, v_cache_ptrs, k_tree_ptrs, v_tree_ptrs, **kw)()


def prepare_kv_commit(k_cache_ptrs: torch.Tensor, v_cache_ptrs: torch.Tensor,
                      k_tree_ptrs: torch.Tensor, v_tree_ptrs: torch.Tensor, *,
                      num_kv_heads: int, head_dim: int, cache_head_stride: int,
                      cache_token_stride: int, tree_row_stride: int, tree_head_stride: int,
                      row_offset: torch.Tensor, keep_rows: torch.Tensor, keep_len: torch.Tensor,
                      prefix_start: torch.Tensor, lengths: torch.Tensor, capacity: int,
                      status: torch.Tensor | None = None) -> PreparedCall:
    """Scatter the kept rows of every layer into the cache, validated and
    bound (call it to run; every run advances ``lengths`` again).

    ``*_ptrs`` are int64 device arrays of per-layer base addresses (see
    pointer_array); keep_rows [n, keep_stride] i32, keep_len [n] i32,
    prefix_start [n] i64, lengths [n] i32 (advanced in place).
    """
    _check_device_tensors((k_cache_ptrs, v_cache_ptrs, k_tree_ptrs, v_tree_ptrs, prefix_start),
                          ("k_cache_ptrs", "v_cache_ptrs", "k_tree_ptrs", "v_tree_ptrs",
                           "prefix_start"), torch.int64)
    _check_device_tensors((row_offset, keep_rows, keep_len, lengths),
                          ("row_offset", "keep_rows", "keep_len", "lengths"), torch.int32)
    layers = k_cache_ptrs.numel()
    _require(v_cache_ptrs.numel() == layers and k_tree_ptrs.numel() == layers
             and v_tree_ptrs.numel() == layers, "per-layer pointer arrays disagree")
    _require(keep_rows.dim() == 2 and keep_rows.is_contiguous(), "keep_rows must be [n, stride]")
    n, keep_stride = keep_rows.shape
    _require(keep_len.numel() == n and lengths.numel() == n and prefix_start.numel() == n
             and row_offset.numel() == n + 1, "request metadata sizes disagree")
    if status is not None:
        _check_device_tensor(status, "status", torch.int32)
    # Positional, in the order of SgKvCommitArgs' fields.
    a = _lib.SgKvCommitArgs(
        layers, n, num_kv_heads, head_dim,
        k_cache_ptrs.data_ptr(), v_cache_ptrs.data_ptr(), cache_head_stride, cache_token_stride,
        k_tree_ptrs.data_ptr(), v_tree_ptrs.data_ptr(), tree_row_stride, tree_head_stride,
        row_offset.data_ptr(), keep_rows.data_ptr(), keep_stride, keep_len.data_ptr(),
        prefix_start.data_ptr(), lengths.data_ptr(), capacity,
        status.data_ptr() if status is not None else 0)
    keep = (k_cache_ptrs, v_cache_ptrs, k_tree_ptrs, v_tree_ptrs, row_offset, keep_rows,
            keep_len, prefix_start, lengths, status)
    return PreparedCall("sg_kv_commit", a, keep)


def kv_split(k_prefix_ptrs: torch.Tensor, v_prefix_ptrs: torch.Tensor,
             k_tree_ptrs: torch.Tensor, v_tree_ptrs: torch.Tensor,
             k_out_ptrs: torch.Tensor, v_out_ptrs: torch.Tensor, *,
             num_kv_heads: int, head_dim: int, prefix_head_stride: int,
             prefix_token_stride: int, tree_row_stride: int, tree_head_stride: int,
             out_head_stride: int, out_token_stride: int, cache_offset: torch.Tensor,
             old_length: torch.Tensor, row_offset: torch.Tensor, keep_rows: torch.Tensor,
             keep_len: torch.Tensor, out_offset: torch.Tensor, max_tokens: int,
             status: torch.Tensor | None = None) -> None:
    """Rebuild every request's cache (old prefix + kept rows) from one packed
    wave, all layers in one call (the non-persistent split).

    ``*_ptrs`` are int64 device arrays of per-layer bases (see pointer_array);
    cache_offset/out_offset [n] i64, old_length/keep_len [n] i32, row_offset
    [n+1] i32, keep_rows [n, keep_stride] i32.
    """
    for t, name in ((k_prefix_ptrs, "k_prefix_ptrs"), (v_prefix_ptrs, "v_prefix_ptrs"),
                    (k_tree_ptrs, "k_tree_ptrs"), (v_tree_ptrs, "v_tree_ptrs"),
                    (k_out_ptrs, "k_out_ptrs"), (v_out_ptrs, "v_out_ptrs"),
                    (cache_offset, "cache_offset"), (out_offset, "out_offset")):
        _check_device_tensor(t, name, torch.int64)
    for t, name in ((old_length, "old_length"), (row_offset, "row_offset"),
                    (keep_rows, "keep_rows"), (keep_len, "keep_len")):
        _check_device_tensor(t, name, torch.int32)
    layers = k_prefix_ptrs.numel()
    _require(all(t.numel() == layers for t in (v_prefix_ptrs, k_tree_ptrs, v_tree_ptrs,
                                               k_out_ptrs, v_out_ptrs)),
             "per-layer pointer arrays disagree")
    _require(keep_rows.dim() == 2 and keep_rows.is_contiguous(), "keep_rows must be [n, stride]")
    n = keep_rows.shape[0]
    _require(cache_offset.numel() == n and out_offset.numel() == n and old_length.numel() == n
             and keep_len.numel() == n and row_offset.numel() == n + 1,
             "request metadata sizes disagree")
    if status is not None:
        _check_device_tensor(status, "status", torch.int32)
    a = _lib.SgKvSplitArgs()
    a.num_layers = layers
    a.num_requests = n
    a.num_kv_heads = num_kv_heads
    a.head_dim = head_dim
    a.max_tokens = max_tokens
    a.keep_stride = keep_rows.shape[1]
    a.k_prefix_layers_dev = k_prefix_ptrs.data_ptr()
    a.v_prefix_layers_dev = v_prefix_ptrs.data_ptr()
    a.prefix_head_stride, a.prefix_token_stride = prefix_head_stride, prefix_token_stride
    a.k_tree_layers_dev = k_tree_ptrs.data_ptr()
    a.v_tree_layers_dev = v_tree_ptrs.data_ptr()
    a.tree_row_stride, a.tree_head_stride = tree_row_stride, tree_head_stride
    a.k_out_layers_dev = k_out_ptrs.data_ptr()
    a.v_out_layers_dev = v_out_ptrs.data_ptr()
    a.out_head_stride, a.out_token_stride = out_head_stride, out_token_stride
    a.cache_offset_dev = cache_offset.data_ptr()
    a.old_length_dev = old_length.data_ptr()
    a.row_offset_dev = row_offset.data_ptr()
    a.keep_rows_dev = keep_rows.data_ptr()
    a.keep_len_dev = keep_len.data_ptr()
    a.out_offset_dev = out_offset.data_ptr()
    a.status_dev = status.data_ptr() if status is not None else 0
    _lib.check(_lib.load().sg_kv_split(ctypes.byref(a), _stream_handle()), "sg_kv_split")


# --------------------------------------------------------------------------
# (C) tree sampling
# --------------------------------------------------------------------------

@dataclass
class SampleResult:
    accept_nodes: torch.Tensor  # [n, max_depth] i32, -1 padded
    accept_len: torch.Tensor    # [n] i32
    bonus: torch.Tensor         # [n] i32
    keep_rows: torch.Tensor     # [n, max_depth + 1] i32 ([0] + nodes, -1 padded)
    row_max: torch.Tensor       # [R] f32
    row_sum: torch.Tensor       # [R] f32
    status: torch.Tensor        # [1] i32
    workspace: torch.Tensor | None = None  # per-slab complement totals of the exit rows


_LOGITS_DTYPES = {torch.float32: _lib.SG_DTYPE_F32, torch.bfloat16: _lib.SG_DTYPE_BF16,
                  torch.float16: _lib.SG_DTYPE_F16}


def _new_status(work: int, device) -> torch.Tensor:
    """A call's status word.  The call writes it when it has work (requests or
    rows), so no fill kernel runs first."""
    make = torch.empty if work > 0 else torch.zeros
    return make(1, dtype=torch.int32, device=device)


def _check_logits(logits: torch.Tensor) -> int:
    _require(isinstance(logits, torch.Tensor) and logits.is_cuda,
             "logits must be a HIP device tensor")
    _require(logits.dtype in _LOGITS_DTYPES,
             f"logits must be float32, bfloat16 or float16, got {logits.dtype}")
    _require(logits.dim() == 2 and logits.stride(1) == 1, "logits must be [R, V] row-contiguous")
    return _LOGITS_DTYPES[logits.dtype]


def _check_sample_out(out: "SampleResult", n: int, rows: int, max_depth: int) -> None:
    """Caller-supplied outputs must fit this call exactly (the kernels index
    them by n, R and max_depth)."""
    expect = {
        "accept_nodes": ((n, max(max_depth, 1)), torch.int32),
        "accept_len": ((n,), torch.int32),
        "bonus": ((n,), torch.int32),
        "keep_rows": ((n, max_depth + 1), torch.int32),
        "row_max": ((rows,), torch.float32),
        "row_sum": ((rows,), torch.float32),
        "status": ((1,), torch.int32),
    }
    for name, (shape, dtype) in expect.items():
        t = getattr(out, name)
        _check_device_tensor(t, f"out.{name}", dtype)
        _require(tuple(t.shape) == shape and t.is_contiguous(),
                 f"out.{name} must be a contiguous {list(shape)} tensor for this call, "
                 f"got {list(t.shape)}")


def _check_sample_inputs(logits, row_offset, parent, token, uniforms, max_depth):
    _check_logits(logits)
    for t, name in ((row_offset, "row_offset"), (parent, "parent"), (token, "token")):
        _check_device_tensor(t, name, torch.int32)
        _require(t.is_contiguous(), f"{name} must be contiguous")
    _check_device_tensor(uniforms, "uniforms", torch.float32)
    _require(uniforms.dim() == 2 and uniforms.is_contiguous(), "uniforms must be [n, U]")
    n = row_offset.numel() - 1
    rows = logits.shape[0]
    _require(uniforms.shape[0] == n, "one uniform row per request")
    _require(uniforms.shape[1] >= 2 * (max_depth + 1), "uniforms must cover 2*(max_depth+1)")
    _require(parent.numel() >= rows and token.numel() >= rows, "parent/token must cover R rows")
    return n, rows


def _sample_args(logits, row_offset, parent, token, uniforms, max_depth, out, n, rows,
                 workspace) -> "_lib.SgTreeSampleArgs":
    a = _lib.SgTreeSampleArgs()
    a.num_requests = n
    a.num_rows = rows
    a.vocab = logits.shape[1]
    a.max_depth = max_depth
    a.logits_dtype = _LOGITS_DTYPES[logits.dtype]
    a.logits_dev = logits.data_ptr()
    a.logits_row_stride = logits.stride(0)
    a.row_offset_dev = row_offset.data_ptr()
    a.parent_dev = parent.data_ptr()
    a.token_dev = token.data_ptr()
    a.uniforms_dev = uniforms.data_ptr()
    a.uniform_stride = uniforms.shape[1]
    a.row_max_dev = out.row_max.data_ptr() if hasattr(out, "row_max") else 0
    a.row_sum_dev = out.row_sum.data_ptr() if hasattr(out, "row_sum") else 0
    a.num_logits_rows = logits.shape[0]
    a.accept_nodes_dev = out.accept_nodes.data_ptr()
    a.accept_len_dev = out.accept_len.data_ptr()
    a.bonus_dev = out.bonus.data_ptr()
    a.keep_rows_dev = out.keep_rows.data_ptr()
    a.status_dev = out.status.data_ptr()
    a.workspace_dev = workspace.data_ptr() if workspace is not None else 0
    a.workspace_bytes = workspace.numel() if workspace is not None else 0
    return a


def tree_sample(logits: torch.Tensor, row_offset: torch.Tensor, parent: torch.Tensor,
                token: torch.Tensor, uniforms: torch.Tensor, max_depth: int,
                out: SampleResult | None = None) -> SampleResult:
    """Temperature-1 tree rejection sampling over all packed rows.

    logits [R, V] fp32, bf16 or f16 (row-contiguous; the 16-bit types widen to
    fp32 exactly), row_offset [n+1] i32 with row_offset[n] == R, parent/token
    [R] i32 (request-local parents, -1 for roots), uniforms [n, U] fp32 with
    U >= 2*(max_depth+1).  ``out`` (optional) must have been made for the same
    n, R and max_depth; its status word is cleared by the call.
    """
    n, rows = _check_sample_inputs(logits, row_offset, parent, token, uniforms, max_depth)
    dev = logits.device
    if out is None:
        depth_slots = max(max_depth, 1)
        out = SampleResult(
            accept_nodes=torch.empty((n, depth_slots), dtype=torch.int32, device=dev),
            accept_len=torch.empty(n, dtype=torch.int32, device=dev),
            bonus=torch.empty(n, dtype=torch.int32, device=dev),
            keep_rows=torch.empty((n, max_depth + 1), dtype=torch.int32, device=dev),
            row_max=torch.empty(rows, dtype=torch.float32, device=dev),
            row_sum=torch.empty(rows, dtype=torch.float32, device=dev),
            status=_new_status(n, dev),
        )
    else:
        _check_sample_out(out, n, rows, max_depth)
    # statistics of every logits row, with their slab pairs in the workspace
    ws_bytes = int(_lib.load().sg_tree_sample_workspace_bytes(n, logits.shape[0],
                                                              logits.shape[1]))
    if out.workspace is None or out.workspace.numel() < ws_bytes:
        out.workspace = torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=dev)
    a = _sample_args(logits, row_offset, parent, token, uniforms, max_depth, out, n, rows,
                     out.workspace)
    _lib.check(_lib.load().sg_tree_sample(ctypes.byref(a), _stream_handle()), "sg_tree_sample")
    return out


def tree_sample_noalloc(logits: torch.Tensor, row_offset: torch.Tensor, parent: torch.Tensor,
                        token: torch.Tensor, uniforms: torch.Tensor, max_depth: int,
                        out: SampleResult) -> SampleResult:
    """tree_sample through sg_tree_sample_noalloc: no device memory is
    allocated (the library's static per-GPU scratch replaces the workspace);
    the caller supplies every output in ``out`` (its ``workspace`` is unused)."""
    n, rows = _check_sample_inputs(logits, row_offset, parent, token, uniforms, max_depth)
    _require(isinstance(out, SampleResult), "sg_tree_sample_noalloc needs caller-owned outputs")
    _check_sample_out(out, n, rows, max_depth)
    a = _sample_args(logits, row_offset, parent, token, uniforms, max_depth, out, n, rows, None)
    _lib.check(_lib.load().sg_tree_sample_noalloc(ctypes.byref(a), _stream_handle()),
               "sg_tree_sample_noalloc")
    return out


@dataclass
class ProjectedSampleResult:
    accept_nodes: torch.Tensor   # [n, max_depth] i32, -1 padded
    accept_len: torch.Tensor     # [n] i32
    bonus: torch.Tensor          # [n] i32, -1 where the walk ended at an unprojected leaf
    keep_rows: torch.Tensor      # [n, max_depth + 1] i32
    terminal_leaf: torch.Tensor  # [n] i32: that leaf's local node id, else -1
    status: torch.Tensor         # [1] i32
    workspace: torch.Tensor


def tree_sample_projected(logits: torch.Tensor, row_offset: torch.Tensor, parent: torch.Tensor,
                          token: torch.Tensor, uniforms: torch.Tensor, max_depth: int, *,
                          row_max: torch.Tensor, row_sum: torch.Tensor,
                          row_map: torch.Tensor | None = None) -> ProjectedSampleResult:
    """The tree walk over LM-head logits whose statistics are already known
    (``lm_head`` wrote them): sg_tree_sample with SG_SAMPLE_STATS_READY.

    ``logits`` [Rp, V] holds the projected rows; ``row_map`` [R] i32 gives
    each packed node's logits row, -1 for a node that was not projected (only
    nodes without children; a walk that ends there reports it in
    ``terminal_leaf`` and leaves its bonus -1), None when row r is node r.
    ``row_max``/``row_sum`` [Rp] f32 are the LM head's row statistics.
    """
    _check_logits(logits)
    for t, name in ((row_offset, "row_offset"), (parent, "parent"), (token, "token")):
        _check_device_tensor(t, name, torch.int32)
        _require(t.is_contiguous(), f"{name} must be contiguous")
    _check_device_tensor(uniforms, "uniforms", torch.float32)
    _require(uniforms.dim() == 2 and uniforms.is_contiguous(), "uniforms must be [n, U]")
    n = row_offset.numel() - 1
    rows = parent.numel()
    logit_rows = logits.shape[0]
    _require(uniforms.shape[0] == n, "one uniform row per request")
    _require(uniforms.shape[1] >= 2 * (max_depth + 1), "uniforms must cover 2*(max_depth+1)")
    _require(token.numel() == rows, "parent and token must both cover the R packed rows")
    for t, name in ((row_max, "row_max"), (row_sum, "row_sum")):
        _check_device_tensor(t, name, torch.float32)
        _require(t.numel() == logit_rows and t.is_contiguous(), f"{name} must be [Rp]")
    if row_map is None:
        _require(logit_rows == rows, "without a row map the logits rows are the packed rows")
    else:
        _check_device_tensor(row_map, "row_map", torch.int32)
        _require(row_map.numel() == rows and row_map.is_contiguous(), "row_map must be [R]")
    dev = logits.device
    depth_slots = max(max_depth, 1)
    ws_bytes = int(_lib.load().sg_tree_sample_workspace_bytes(n, 0, logits.shape[1]))
    out = ProjectedSampleResult(
        accept_nodes=torch.empty((n, depth_slots), dtype=torch.int32, device=dev),
        accept_len=torch.empty(n, dtype=torch.int32, device=dev),
        bonus=torch.empty(n, dtype=torch.int32, device=dev),
        keep_rows=torch.empty((n, max_depth + 1), dtype=torch.int32, device=dev),
        terminal_leaf=torch.empty(n, dtype=torch.int32, device=dev),
        status=_new_status(n, dev),
        workspace=torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=dev))
    a = _sample_args(logits, row_offset, parent, token, uniforms, max_depth, out, n, rows,
                     out.workspace)
    a.row_max_dev = row_max.data_ptr()
    a.row_sum_dev = row_sum.data_ptr()
    a.logits_row_dev = row_map.data_ptr() if row_map is not None else 0
    a.num_logits_rows = logit_rows
    a.flags = _lib.SG_SAMPLE_STATS_READY
    a.terminal_leaf_dev = out.terminal_leaf.data_ptr()
    _lib.check(_lib.load().sg_tree_sample(ctypes.byref(a), _stream_handle()), "sg_tree_sample")
    return out


def row_stats(logits: torch.Tensor):
    dtype = _check_logits(logits)
    rows = logits.shape[0]
    m = torch.empty(rows, dtype=torch.float32, device=logits.device)
    z = torch.empty(rows, dtype=torch.float32, device=logits.device)
    _lib.check(_lib.load().sg_row_stats(logits.data_ptr(), dtype, logits.stride(0),
                                        logits.shape[1], rows, m.data_ptr(), z.data_ptr(),
                                        _stream_handle()),
               "sg_row_stats")
    return m, z


def exp_probe(x: torch.Tensor) -> torch.Tensor:
    _check_device_tensor(x, "x", torch.float32)
    x = x.contiguous()
    out = torch.empty_like(x)
    _lib.check(_lib.load().sg_exp_probe(x.data_ptr(), out.data_ptr(), x.numel(),
                                        _stream_handle()), "sg_exp_probe")
    return out


class ClockProbe:
    """Average shader clock over timed regions, per XCD.

    ``mark()`` enqueues ``sg_clock_probe`` on the current stream and returns
    the mark's index; after the stream has been synchronized, ``ghz(a, b)``
    gives {xcd: GHz} between marks ``a`` and ``b``.  The shader-cycle counters
    of different CUs are not aligned, so every CU that both marks saw gives
    its own clock (its counter's delta over the constant-rate counter's delta,
    times that counter's rate) and each XCD reports the median over its CUs.
    ``blocks`` workgroups per mark (1,024: every CU is seen by nearly every
    mark).  ``spread(a)`` is the largest difference of the shader-cycle
    counter between workgroups on one CU at one mark.
    """

    def __init__(self, device, capacity: int = 512, blocks: int = 1024):
        lib = _lib.load()
        index = torch.device(device).index or 0
        khz = int(lib.sg_wall_clock_khz(index))
        _require(khz > 0, "sg_wall_clock_khz failed: "
                 + lib.sg_last_error().decode(errors="replace"))
        self.wall_hz = khz * 1e3
        self.blocks, self.capacity, self.count = blocks, capacity, 0
        self._buf = torch.zeros((capacity, blocks, 4), dtype=torch.int64, device=device)

    def mark(self) -> int:
        _require(self.count < self.capacity, "clock probe capacity exhausted")
        _lib.check(_lib.load().sg_clock_probe(self._buf[self.count].data_ptr(), self.blocks,
                                              _stream_handle()), "sg_clock_probe")
        self.count += 1
        return self.count - 1

    def _per_cu(self, mark: int) -> dict:
        h = self._buf[mark].cpu().numpy()
        keys = h[:, 0] * 256 + ((h[:, 3] >> 8) & 0xFF)  # XCD, engine, array, CU
        return {int(k): (np.median(h[keys == k][:, 1]), np.median(h[keys == k][:, 2]),
                         int(np.ptp(h[keys == k][:, 1])))
                for k in np.unique(keys)}

    def ghz(self, a: int, b: int) -> dict:
        ra, rb = self._per_cu(a), self._per_cu(b)
        per_xcd: dict = {}
        for k in ra.keys() & rb.keys():
            ticks = rb[k][1] - ra[k][1]
            if ticks > 0:
                per_xcd.setdefault(k // 256, []).append(
                    (rb[k][0] - ra[k][0]) / ticks * self.wall_hz / 1e9)
        return {x: float(np.median(v)) for x, v in sorted(per_xcd.items())}

    def spread(self, a: int) -> int:
        return max(v[2] for v in self._per_cu(a).values())


# --------------------------------------------------------------------------
# (D) LM head with fused statistics
# --------------------------------------------------------------------------

@dataclass
class LmHeadResult:
    logits: torch.Tensor      # [Rp, V] bf16 (a view of rows padded to 8 elements)
    tile_stats: torch.Tensor  # [Rp, ceil(V/128), 2] f32: (max, sum of E(x - max)) per tile
    row_max: torch.Tensor     # [Rp] f32
    row_sum: torch.Tensor     # [Rp] f32
    status: torch.Tensor      # [1] i32: SG_EINVAL when a row index was out of range


class PackedLmHead:
    """``lm_head.weight`` re-laid out once for ``sg_lm_head_packed`` (every
    16 KiB weight stage of the kernel contiguous).  Holds the packed bytes
    beside the model's own weight; ``shape`` and ``dtype`` are the original
    weight's, so it stands in for it wherever ``lm_head`` takes a weight."""
    __slots__ = ("packed", "shape", "dtype", "device")

    def __init__(self, weight: torch.Tensor):
        _check_device_tensor(weight, "weight", torch.bfloat16)
        _require(weight.dim() == 2 and weight.stride(1) == 1,
                 "weight must be a row-contiguous matrix")
        vocab, hsize = weight.shape
        lib = _lib.load()
        nbytes = int(lib.sg_lm_head_packed_bytes(vocab, hsize))
        _require(nbytes > 0, "weight size unsupported (H a positive multiple of 64)")
        self.packed = torch.empty(nbytes // 2, dtype=torch.bfloat16, device=weight.device)
        _lib.check(lib.sg_lm_head_pack_weight(weight.data_ptr(), weight.stride(0), vocab, hsize,
                                              self.packed.data_ptr(), _stream_handle()),
                   "sg_lm_head_pack_weight")
        self.shape = torch.Size((vocab, hsize))
        self.dtype = weight.dtype
        self.device = weight.device


def pack_lm_head(weight: torch.Tensor) -> PackedLmHead:
    """One-time packing of ``lm_head.weight`` for ``lm_head`` (enqueued on
    torch's current stream)."""
    return PackedLmHead(weight)


def lm_head(hidden: torch.Tensor, weight,
            row_index: torch.Tensor | None = None) -> LmHeadResult:
    """bf16 logits of the selected hidden rows and their softmax statistics
    (sg_lm_head, or sg_lm_head_packed for a PackedLmHead).

    ``hidden`` [N, H] bf16 (row-contiguous, H a multiple of 64), ``weight``
    [V, H] bf16 (``lm_head.weight``) or its ``PackedLmHead`` (same results,
    bit for bit), ``row_index`` [Rp] i32 selects the rows
    to project (None: all N).  Replaces ``lm_head(hidden)`` +
    ``probabilities(...)`` on the rows a tree walk can need
    (fused_tree_sampling.py:2899-2913, :2974-2984).
    """
    packed = isinstance(weight, PackedLmHead)
    checked = (hidden,) if packed else (hidden, weight)
    for t, name in zip(checked, ("hidden", "weight")):
        _check_device_tensor(t, name, torch.bfloat16)
        _require(t.dim() == 2 and t.stride(1) == 1, f"{name} must be a row-contiguous matrix")
    _require(hidden.shape[1] == weight.shape[1], "hidden and weight disagree on the hidden size")
    if row_index is not None:
        _check_device_tensor(row_index, "row_index", torch.int32)
        _require(row_index.dim() == 1 and row_index.is_contiguous(), "row_index must be [Rp]")
    rows = row_index.numel() if row_index is not None else hidden.shape[0]
    vocab, hsize = weight.shape
    dev = hidden.device
    pad = (vocab + 7) // 8 * 8
    tiles = int(_lib.load().sg_lm_head_tile_count(vocab))
    logits = torch.empty((rows, pad), dtype=torch.bfloat16, device=dev)
    res = LmHeadResult(
        logits=logits[:, :vocab],
        tile_stats=torch.empty((rows, tiles, 2), dtype=torch.float32, device=dev),
        row_max=torch.empty(rows, dtype=torch.float32, device=dev),
        row_sum=torch.empty(rows, dtype=torch.float32, device=dev),
        status=_new_status(rows, dev))
    a = _lib.SgLmHeadArgs()
    a.num_rows = rows
    a.hidden_size = hsize
    a.vocab = vocab
    a.num_hidden_rows = hidden.shape[0]
    a.hidden_dev = hidden.data_ptr()
    a.hidden_row_stride = hidden.stride(0)
    a.row_index_dev = row_index.data_ptr() if row_index is not None else 0
    a.weight_dev = weight.packed.data_ptr() if packed else weight.data_ptr()
    a.weight_row_stride = hsize if packed else weight.stride(0)
    a.logits_dev = logits.data_ptr()
    a.logits_row_stride = pad
    a.tile_stats_dev = res.tile_stats.data_ptr()
    a.row_max_dev = res.row_max.data_ptr()
    a.row_sum_dev = res.row_sum.data_ptr()
    a.status_dev = res.status.data_ptr()
    _lib.check(_lib.load().sg_lm_head_fresh(ctypes.byref(a), int(packed), _stream_handle()),
               "sg_lm_head_packed" if packed else "sg_lm_head")
    return res


# --------------------------------------------------------------------------
# (E) the cache in 4 bits
# --------------------------------------------------------------------------
# Rows of D values as codes [..., D/2] and scales [..., D/32] (uint8): e2m1
# elements, two a byte, with one power-of-two scale for 32 of them (the header
# says which).  Every value is a bf16 value.

def _check_mx4(codes: torch.Tensor, scales: torch.Tensor, name: str) -> None:
    _check_device_tensor(codes, f"{name}_codes", torch.uint8)
    _check_device_tensor(scales, f"{name}_scales", torch.uint8)
    _require(codes.dim() >= 2 and codes.shape[:-1] == scales.shape[:-1]
             and codes.shape[-1] == 16 * scales.shape[-1] and scales.shape[-1] >= 1,
             f"{name}_codes must be [..., tokens, D/2] and {name}_scales [..., tokens, D/32]")
    _require(codes.stride(-1) == 1 and scales.stride(-1) == 1,
             f"{name}_codes and {name}_scales must have a contiguous last dimension")


def tree_attention_mx4(q: torch.Tensor, k_codes: torch.Tensor, k_scales: torch.Tensor,
                       v_codes: torch.Tensor, v_scales: torch.Tensor, k_tree: torch.Tensor,
                       v_tree: torch.Tensor, row_offset: torch.Tensor,
                       prefix_start: torch.Tensor, prefix_len: torch.Tensor,
                       parent: torch.Tensor, plan: AttnPlan, out: torch.Tensor | None = None,
                       scale: float | None = None,
                       status: torch.Tensor | None = None) -> torch.Tensor:
    """Packed tree attention of one layer over a 4-bit cache (see
    prepare_tree_attention_mx4)."""
    args, out, _ = _mx4_attention_args(q, k_codes, k_scales, v_codes, v_scales, k_tree, v_tree,
                                       row_offset, prefix_start, prefix_len, parent, plan, out,
                                       scale, status)
    _lib.check(_lib.load().sg_tree_attn_mx4_fwd(ctypes.byref(args), _stream_handle()),
               "sg_tree_attn_mx4_fwd")
    return out


def prepare_tree_attention_mx4(q: torch.Tensor, k_codes: torch.Tensor, k_scales: torch.Tensor,
                               v_codes: torch.Tensor, v_scales: torch.Tensor,
                               k_tree: torch.Tensor, v_tree: torch.Tensor,
                               row_offset: torch.Tensor, prefix_start: torch.Tensor,
                               prefix_len: torch.Tensor, parent: torch.Tensor, plan: AttnPlan,
                               out: torch.Tensor | None = None, scale: float | None = None,
                               status: torch.Tensor | None = None) -> PreparedCall:
    """Packed tree attention of one layer whose prefixes are held in 4 bits,
    validated and bound (call it to run).

    k/v_codes [Hkv, tokens, D/2] and k/v_scales [Hkv, tokens, D/32] uint8 (the
    layer's arena, rows written by ``kv_commit_mx4``); everything else, the plan
    included, as in ``prepare_tree_attention``.  What lies behind a request's
    last token is not looked at.  An infinity or a NaN in a tree row reaches only
    the rows that see it; a cached row packed from one gives NaN.  ``scale`` (positive,
    finite; head_dim ** -0.5 without it) is checked by the call itself.
    """
    args, out, run = _mx4_attention_args(q, k_codes, k_scales, v_codes, v_scales, k_tree, v_tree,
                                         row_offset, prefix_start, prefix_len, parent, plan, out,
                                         scale, status)
    keep = (q, k_codes, k_scales, v_codes, v_scales, k_tree, v_tree, row_offset, prefix_start,
            prefix_len, parent, run.device, run.host, run.workspace, out, status)
    return PreparedCall("sg_tree_attn_mx4_fwd", args, keep, result=out)


def _explain_mx4_attention(q, k_codes, k_scales, v_codes, v_scales, k_tree, v_tree, row_offset,
                           prefix_start, prefix_len, parent, plan, out, status) -> None:
    """Raise ValueError for the first argument that does not fit."""
    for t, name in ((q, "q"), (k_tree, "k_tree"), (v_tree, "v_tree")):
        _check_rows(t, name)
    _check_mx4(k_codes, k_scales, "k")
    _check_mx4(v_codes, v_scales, "v")
    _check_device_tensors((row_offset, prefix_len, parent),
                          ("row_offset", "prefix_len", "parent"), torch.int32)
    _check_device_tensor(prefix_start, "prefix_start", torch.int64)
    for t, name in ((row_offset, "row_offset"), (prefix_len, "prefix_len"), (parent, "parent"),
                    (prefix_start, "prefix_start")):
        _require(t.is_contiguous(), f"{name} must be contiguous")
    _require(q.dim() == 3 and k_tree.dim() == 3 and k_codes.dim() == 3,
             "q/k_tree must be [R, H, D] and k_codes [Hkv, tokens, D/2]")
    _require(k_codes.shape == v_codes.shape and k_codes.stride() == v_codes.stride()
             and k_scales.stride() == v_scales.stride(),
             "k and v codes and scales must share shape and strides")
    _require(k_codes.shape[2] * 2 == q.shape[2], "head dims disagree")
    _require(not any((t.data_ptr() | t.stride(0) | t.stride(1)) % 16 for t in (k_codes, v_codes)),
             "codes must be 16-byte aligned, their strides multiples of 16 bytes")
    _require(k_tree.shape == (q.shape[0], k_codes.shape[0], q.shape[2])
             and v_tree.shape == k_tree.shape and k_tree.stride() == v_tree.stride(),
             "k_tree/v_tree must be [R, Hkv, D] with equal strides")
    _require(plan.device is not None and plan.device.is_cuda, "plan is not on the device")
    _require(parent.numel() >= q.shape[0], "parent must cover every packed row")
    _require(row_offset.numel() == prefix_len.numel() + 1
             and prefix_start.numel() == prefix_len.numel(),
             "request metadata sizes disagree")
    if status is not None:
        _check_device_tensor(status, "status", torch.int32)
    if out is not None:
        _check_rows(out, "out")
        _require(out.shape == q.shape, "out must be [R, Hq, D]")
    for t, name in ((k_codes, "k_codes"), (k_scales, "k_scales"), (v_codes, "v_codes"),
                    (v_scales, "v_scales"), (k_tree, "k_tree"), (v_tree, "v_tree"),
                    (row_offset, "row_offset"), (prefix_start, "prefix_start"),
                    (prefix_len, "prefix_len"), (parent, "parent"), (out, "out"),
                    (status, "status"), (plan.device, "plan")):
        _require(t is None or t.device == q.device, f"{name} must be on q's device")
    _check_current(q, "q")


def _mx4_attention_args(q, k_codes, k_scales, v_codes, v_scales, k_tree, v_tree, row_offset,
                        prefix_start, prefix_len, parent, plan, out, scale, status):
    """The call's argument struct and output, of arguments that fit, and the plan that
    it runs.

    A call takes a few microseconds on the GPU at the least, so everything is
    looked at once here; what is wrong is found out by _explain_mx4_attention."""
    try:
        bf16, u8, i32 = torch.bfloat16, torch.uint8, torch.int32
        rows, hq, dim = q.shape
        hkv, tokens, half = k_codes.shape
        qs, cs, ss, ts = q.stride(), k_codes.stride(), k_scales.stride(), k_tree.stride()
        at = (q.data_ptr(), k_codes.data_ptr(), v_codes.data_ptr(), k_tree.data_ptr(),
              v_tree.data_ptr())
        n = prefix_len.numel()
        device = q.get_device()  # -1 on the CPU
        kv = (hkv, tokens, half // 16)
        fits = True
        if out is not None:
            os = out.stride()
            fits = (out.dtype == bf16 and out.shape == q.shape and os[2] == 1
                    and not (os[0] | os[1]) & 7 and not out.data_ptr() & 15
                    and out.get_device() == device)
        if status is not None:
            fits = fits and status.dtype == i32 and status.get_device() == device
        fits = (
            fits and q.dtype == bf16 and k_tree.dtype == bf16 and v_tree.dtype == bf16
            and k_codes.dtype == u8 and k_scales.dtype == u8 and v_codes.dtype == u8
            and v_scales.dtype == u8 and row_offset.dtype == i32 and prefix_len.dtype == i32
            and parent.dtype == i32 and prefix_start.dtype == torch.int64
            and 2 * half == dim and v_codes.shape == k_codes.shape
            and v_scales.shape == kv and k_scales.shape == kv
            and k_tree.shape == (rows, hkv, dim) and v_tree.shape == k_tree.shape
            and v_codes.stride() == cs and v_scales.stride() == ss and v_tree.stride() == ts
            and qs[2] == 1 and cs[2] == 1 and (ss[2] == 1 or half == 16) and ts[2] == 1
            and not (at[0] | at[1] | at[2] | at[3] | at[4] | cs[0] | cs[1]) & 15
            and not (qs[0] | qs[1] | ts[0] | ts[1]) & 7
            and row_offset.numel() == n + 1 and prefix_start.numel() == n
            and parent.numel() >= rows and row_offset.is_contiguous()
            and prefix_len.is_contiguous() and parent.is_contiguous()
            and prefix_start.is_contiguous()
            and device == torch.cuda.current_device()
            and k_codes.get_device() == device and k_scales.get_device() == device
            and v_codes.get_device() == device and v_scales.get_device() == device
            and k_tree.get_device() == device and v_tree.get_device() == device
            and row_offset.get_device() == device and prefix_len.get_device() == device
            and parent.get_device() == device and prefix_start.get_device() == device
            and plan.device is not None and plan.device.get_device() == device)
    except (AttributeError, TypeError, ValueError, RuntimeError):  # no tensors, no GPU
        fits = False
    if not fits:
        _explain_mx4_attention(q, k_codes, k_scales, v_codes, v_scales, k_tree, v_tree,
                               row_offset, prefix_start, prefix_len, parent, plan, out, status)
    _require(fits, "the arguments do not fit together")
    check_plan_call(plan, n, rows, hq, hkv, dim)
    plan = plan.in_mx4()
    if out is None:
        out = torch.empty((rows, hq, dim), dtype=bf16, device=q.device)
        os = out.stride()
    workspace = plan.workspace
    attn = _lib.SgTreeAttnArgs(
        n, rows, hq, hkv, dim, float(dim ** -0.5 if scale is None else scale),
        at[0], qs[0], qs[1], at[1], at[2], cs[0], cs[1], at[3], at[4], ts[0], ts[1],
        row_offset.data_ptr(), prefix_start.data_ptr(), prefix_len.data_ptr(),
        parent.data_ptr(), out.data_ptr(), os[0], os[1],
        plan.device.data_ptr(), plan.host.ctypes.data, plan.units, plan.merges,
        workspace.data_ptr() if workspace is not None else 0,
        workspace.numel() if workspace is not None else 0,
        status.data_ptr() if status is not None else 0)
    return _lib.SgTreeAttnMx4Args(attn, k_scales.data_ptr(), v_scales.data_ptr(), ss[0],
                                  ss[1]), out, plan


def kv_commit_mx4(k_code_ptrs: torch.Tensor, k_scale_ptrs: torch.Tensor,
                  v_code_ptrs: torch.Tensor, v_scale_ptrs: torch.Tensor,
                  k_tree_ptrs: torch.Tensor, v_tree_ptrs: torch.Tensor, **kw) -> None:
    """Pack the kept rows of every layer into the 4-bit cache (one call; see
    prepare_kv_commit_mx4)."""
    prepare_kv_commit_mx4(k_code_ptrs, k_scale_ptrs, v_code_ptrs, v_scale_ptrs, k_tree_ptrs,
                          v_tree_ptrs, **kw)()


def prepare_kv_commit_mx4(k_code_ptrs: torch.Tensor, k_scale_ptrs: torch.Tensor,
                          v_code_ptrs: torch.Tensor, v_scale_ptrs: torch.Tensor,
                          k_tree_ptrs: torch.Tensor, v_tree_ptrs: torch.Tensor, *,
                          num_kv_heads: int, head_dim: int, code_head_stride: int,
                          code_token_stride: int, scale_head_stride: int,
                          scale_token_stride: int, tree_row_stride: int, tree_head_stride: int,
                          row_offset: torch.Tensor, keep_rows: torch.Tensor | None,
                          keep_len: torch.Tensor, prefix_start: torch.Tensor,
                          lengths: torch.Tensor, capacity: int,
                          status: torch.Tensor | None = None) -> PreparedCall:
    """``prepare_kv_commit`` into a 4-bit arena: the kept bf16 rows of every
    layer are packed and appended.

    ``*_ptrs`` are int64 device arrays of per-layer base addresses; the strides of
    codes and scales are in bytes.  ``keep_rows`` [n, keep_stride] i32, or None: a
    request keeps its rows 0 .. keep_len - 1 (a prefilled prompt).  The launch then covers
    ``capacity`` rows a request; ``set(keep_stride=...)`` of the prepared call bounds it
    by the longest prompt, where the host knows that (a longer one reports SG_ERANGE).
    """
    pointers = (k_code_ptrs, k_scale_ptrs, v_code_ptrs, v_scale_ptrs, k_tree_ptrs, v_tree_ptrs)
    names = ("k_code_ptrs", "k_scale_ptrs", "v_code_ptrs", "v_scale_ptrs", "k_tree_ptrs",
             "v_tree_ptrs")
    _check_device_tensors((*pointers, prefix_start), (*names, "prefix_start"), torch.int64)
    _check_device_tensors((row_offset, keep_len, lengths),
                          ("row_offset", "keep_len", "lengths"), torch.int32)
    for t, name in zip((*pointers, prefix_start, row_offset, keep_len, lengths),
                       (*names, "prefix_start", "row_offset", "keep_len", "lengths")):
        _require(t.is_contiguous(), f"{name} must be contiguous")
    layers = k_code_ptrs.numel()
    _require(all(t.numel() == layers for t in pointers), "per-layer pointer arrays disagree")
    n = keep_len.numel()
    keep_stride = max(1, int(capacity))
    if keep_rows is not None:
        _check_device_tensor(keep_rows, "keep_rows", torch.int32)
        _require(keep_rows.dim() == 2 and keep_rows.is_contiguous(),
                 "keep_rows must be [n, stride]")
        _require(keep_rows.shape[0] == n, "request metadata sizes disagree")
        keep_stride = keep_rows.shape[1]
    _require(lengths.numel() == n and prefix_start.numel() == n and row_offset.numel() == n + 1,
             "request metadata sizes disagree")
    if status is not None:
        _check_device_tensor(status, "status", torch.int32)
    _check_current(lengths, "lengths", *pointers, prefix_start, row_offset, keep_len, keep_rows,
                   status)
    a = _lib.SgKvCommitMx4Args(
        layers, n, num_kv_heads, head_dim, *(t.data_ptr() for t in pointers[:4]),
        code_head_stride, code_token_stride, scale_head_stride, scale_token_stride,
        k_tree_ptrs.data_ptr(), v_tree_ptrs.data_ptr(), tree_row_stride, tree_head_stride,
        row_offset.data_ptr(), keep_rows.data_ptr() if keep_rows is not None else 0, keep_stride,
        keep_len.data_ptr(), prefix_start.data_ptr(), lengths.data_ptr(), capacity,
        status.data_ptr() if status is not None else 0)
    keep = (*pointers, row_offset, keep_rows, keep_len, prefix_start, lengths, status)
    return PreparedCall("sg_kv_commit_mx4", a, keep)


def kv_load_mx4(codes: torch.Tensor, scales: torch.Tensor,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """bf16 values [..., tokens, D] of packed rows codes [..., tokens, D/2] and
    scales [..., tokens, D/32] (views of an arena too: the dimensions before the
    last two must be one stride apart)."""
    _check_mx4(codes, scales, "cache")
    dim = 2 * codes.shape[-1]
    shape = (*codes.shape[:-1], dim)
    if out is None:
        out = torch.empty(shape, dtype=torch.bfloat16, device=codes.device)
    _check_rows(out, "out")
    _require(tuple(out.shape) == shape, "out must be [..., tokens, D]")
    if out.numel() == 0:
        return out
    flat = []
    for t, name in ((codes, "codes"), (scales, "scales"), (out, "out")):
        try:
            flat.append(t.view(-1, *t.shape[-2:]))
        except RuntimeError:
            raise ValueError(f"{name}: the dimensions before the last two must be one stride "
                             f"apart") from None
    c, s, o = flat
    _require(not (c.data_ptr() | c.stride(0) | c.stride(1)) % 4,
             "codes must be 4-byte aligned, their strides multiples of 4 bytes")
    _check_current(codes, "codes", scales, out)
    _lib.check(_lib.load().sg_kv_load_mx4(
        c.data_ptr(), c.stride(0), c.stride(1), s.data_ptr(), s.stride(0), s.stride(1),
        c.shape[0], c.shape[1], dim, o.data_ptr(), o.stride(0), o.stride(1), _stream_handle()),
        "sg_kv_load_mx4")
    return out


# --------------------------------------------------------------------------
# (F) projections in 8-bit floating point
# --------------------------------------------------------------------------

FP8_BLOCK = 128  # columns (and weight rows) of a scale


@dataclass
class Fp8Rows:
    """Activation rows in e4m3 with an fp32 scale for each row and 128 columns."""
    codes: torch.Tensor   # [R, K] float8_e4m3fn, a view of rows padded with zeros to 128 columns
    scales: torch.Tensor  # [R, ceil(K/128)] f32, a view of [ceil(K/128), R]

    @property
    def shape(self) -> torch.Size:
        return self.codes.shape

    def dequantize(self) -> torch.Tensor:
        """The values the rows stand for, [R, K] f32."""
        k = self.codes.shape[1]
        return self.codes.float() * self.scales.repeat_interleave(FP8_BLOCK, 1)[:, :k]


def _new_fp8_rows(rows: int, columns: int, device) -> "tuple[Fp8Rows, _lib.SgFp8RowsOut]":
    blocks = (columns + FP8_BLOCK - 1) // FP8_BLOCK
    padded = blocks * FP8_BLOCK
    codes = torch.empty((rows, padded), dtype=torch.float8_e4m3fn, device=device)
    scales = torch.empty_strided((rows, blocks), (1, rows), dtype=torch.float32, device=device)
    out = _lib.SgFp8RowsOut(codes.data_ptr(), padded, scales.data_ptr(), rows)
    return Fp8Rows(codes if padded == columns else codes[:, :columns], scales), out


def _check_current(t: torch.Tensor, name: str, *others: torch.Tensor | None) -> None:
    """t, and whatever else the call is given, on the current device."""
    device = torch.cuda.current_device()
    if t.get_device() != device:
        raise ValueError(f"{name} is on {t.device}, which is not the current device")
    for o in others:
        if o is not None and o.get_device() != device:
            raise ValueError(f"a tensor is on {o.device}, {name} on {t.device}")


def quantize_fp8(x: torch.Tensor) -> Fp8Rows:
    """bf16 rows [R, K] in e4m3 with a scale for each row and 128 columns (K a
    multiple of 8, rows 16-byte aligned)."""
    _check_rows(x, "x")
    _require(x.dim() == 2, "x must be [R, K]")
    _check_current(x, "x")
    count, columns = x.shape
    rows, out = _new_fp8_rows(count, columns, x.device)
    _lib.check(_lib.load().sg_fp8_quantize_rows(x.data_ptr(), x.stride(0), count, columns,
                                                ctypes.byref(out), _stream_handle()),
               "sg_fp8_quantize_rows")
    return rows


def quantize_fp8_weight(weight: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """A weight [N, K] as e4m3 codes [N, K] and fp32 scales [ceil(N/128),
    ceil(K/128)], the largest magnitude of a block at 448.  Once per weight, in
    torch operations, on any device."""
    _require(weight.dim() == 2 and weight.numel() > 0, "weight must be a matrix")
    n, k = weight.shape
    pad = torch.nn.functional.pad(weight.float(), (0, -k % FP8_BLOCK, 0, -n % FP8_BLOCK))
    blocks = pad.unflatten(0, (-1, FP8_BLOCK)).unflatten(-1, (-1, FP8_BLOCK))
    most = blocks.abs().amax((1, 3)).clamp_min(2.0 ** -100)
    codes = (blocks * (448.0 / most)[:, None, :, None]).to(torch.float8_e4m3fn)
    return (codes.flatten(2).flatten(0, 1)[:n, :k].contiguous(), most / 448.0)


class PackedFp8Weight:
    """An e4m3 weight [N, K] and its block scales, re-laid out once for
    ``fp8_matmul`` (the order in which the matrix instruction takes it)."""
    __slots__ = ("packed", "scales", "shape", "device")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        _check_device_tensor(codes, "codes", torch.float8_e4m3fn)
        _require(codes.dim() == 2 and codes.numel() > 0 and codes.stride(1) == 1
                 and codes.stride(0) >= codes.shape[1], "codes must be a row-contiguous matrix")
        _check_device_tensor(scales, "scales", torch.float32)
        n, k = codes.shape
        _require(tuple(scales.shape) == (-(-n // FP8_BLOCK), -(-k // FP8_BLOCK)),
                 "scales must be [ceil(N/128), ceil(K/128)]")
        _require(scales.device == codes.device, "codes and scales must be on one device")
        _check_current(codes, "codes")
        lib = _lib.load()
        nbytes = int(lib.sg_fp8_packed_bytes(n, k))
        _require(nbytes > 0, "weight size unsupported (N and K up to 2^24)")
        self.packed = torch.empty(nbytes, dtype=torch.uint8, device=codes.device)
        self.scales = scales.contiguous().clone()
        self.shape = torch.Size((n, k))
        self.device = codes.device
        _lib.check(lib.sg_fp8_pack_weight(codes.data_ptr(), codes.stride(0), n, k,
                                          self.packed.data_ptr(), _stream_handle()),
                   "sg_fp8_pack_weight")


def pack_fp8_weight(codes: torch.Tensor, scales: torch.Tensor) -> PackedFp8Weight:
    """One-time packing of an e4m3 weight (``quantize_fp8_weight``, or a checkpoint
    with 128 x 128 block scales) for ``fp8_matmul``, enqueued on torch's current
    stream."""
    return PackedFp8Weight(codes, scales)


def fp8_matmul(rows: Fp8Rows, weight: PackedFp8Weight,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """rows @ weight.T in bf16, [R, N]: e4m3 products, fp32 sums, each block of 128
    columns scaled by its row's and its weight block's scale.

    ``out`` (optional) is a bf16 [R, N] tensor with 16-byte aligned rows.  Without
    it the result is a view of rows padded to 8 columns.
    """
    _require(isinstance(rows, Fp8Rows) and isinstance(weight, PackedFp8Weight),
             "fp8_matmul takes Fp8Rows and a PackedFp8Weight")
    codes, scales = rows.codes, rows.scales
    _check_device_tensor(codes, "codes", torch.float8_e4m3fn)
    _check_device_tensor(scales, "scales", torch.float32)
    n, k = weight.shape
    blocks = (k + FP8_BLOCK - 1) // FP8_BLOCK
    _require(codes.dim() == 2 and codes.shape[1] == k, "rows and weight disagree on K")
    count = codes.shape[0]
    device = codes.device
    cs, ss = codes.stride(), scales.stride()
    _require(scales.shape == (count, blocks) and (ss[0] == 1 or count == 1),
             "scales must be the [R, ceil(K/128)] view of the quantized rows")
    _require(codes.get_device() == weight.packed.get_device() == scales.get_device(),
             "rows and weight must be on one device")
    _check_current(codes, "rows")
    # The padded columns behind a row are read: they must be there.
    _require(count == 0 or (cs[1] == 1 and cs[0] >= FP8_BLOCK * blocks
                            and codes.untyped_storage().nbytes() - codes.storage_offset()
                            >= (count - 1) * cs[0] + FP8_BLOCK * blocks),
             "codes must be rows padded with zeros to 128 columns")
    if out is None:
        out = torch.empty((count, (n + 7) // 8 * 8), dtype=torch.bfloat16, device=device)
        if n % 8:
            out = out[:, :n]
    else:
        _check_rows(out, "out")
        _require(tuple(out.shape) == (count, n) and out.device == device,
                 "out must be [R, N] on the rows' device")
    lib = _lib.load()
    nbytes = lib.sg_fp8_matmul_workspace_bytes(count, n, k)
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes > 0 else None
    a = _lib.SgFp8MatmulArgs(
        count, n, k, 0, codes.data_ptr(), cs[0], scales.data_ptr(),
        ss[1] if blocks > 1 else max(count, 1), weight.packed.data_ptr(),
        weight.scales.data_ptr(), out.data_ptr(), out.stride(0),
        workspace.data_ptr() if workspace is not None else 0, max(nbytes, 0))
    _lib.check(lib.sg_fp8_matmul(ctypes.byref(a), _stream_handle()), "sg_fp8_matmul")
    return out
