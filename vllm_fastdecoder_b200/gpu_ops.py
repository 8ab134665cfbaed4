"""Torch-level front end of the sm_100a kernels (the C ABI in include/).

Mirrors the reference operator interface of fastdecode/cpu_ops.py and
fastdecode/csrc/cpu_attn.cpp:
  load_ext()                          -> object with decode_attn / store_kv /
                                         set_num_threads / get_num_threads /
                                         has_avx2, like cpu_ops.load_ext
                                         (cpu_ops.py:21-46)
  decode_attn(q, k_cache, v_cache, block_table, lens, scale, out, lse)
                                      (cpu_attn.cpp:456-489), same argument
                                      meaning and the same RuntimeError
                                      checks (:460-477), on device tensors or
                                      on pinned host caches read over PCIe
  store_kv(k, v, slots, k_cache, v_cache)
                                      (cpu_attn.cpp:492-517), range error ->
                                      RuntimeError (:506-510)
  merge_attn_states(out, o_a, lse_a, o_b, lse_b)
                                      vLLM's op as called at backend.py:54-55
plus the two-tier entry points the backend uses (decode_tiered, store_kv_tiered,
merge_partials), and the operators of a step whose requests bring several new
tokens: extend_tables (block tables, slots and positions from lengths),
rope_store_kv (multi-axis rotary positions with the KV write), chunk_attn (the
new tokens' attention over the cached context of either tier) and cross_attn
(attention to an encoder's states); and of what follows it: verify_drafts
(drafted tokens against the target's probabilities), key_weights, select_keys
and move_keys (a cache cut to the keys that get attention) and trim_tables
(the blocks behind shorter requests given back).  Every call is asynchronous on the current CUDA stream.
There is no CPU path: without the native library or a CUDA device these raise.
"""

from __future__ import annotations

import ctypes
import math
import os
import struct
from dataclasses import dataclass
from functools import lru_cache

import torch

from vllm_fastdecoder_b200 import _native as nat

_DTYPE = {torch.float16: nat.FD_DTYPE_F16, torch.bfloat16: nat.FD_DTYPE_BF16, torch.float32: nat.FD_DTYPE_F32}


def dtype_code(dt: torch.dtype) -> int:
    try:
        return _DTYPE[dt]
    except KeyError:
        raise RuntimeError(f"unsupported dtype {dt}") from None


def _check(cond: bool, msg: str) -> None:
    if not cond:
        raise RuntimeError(msg)


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


# ------------------------------------------------------------- per-device state

_WS: dict[int, torch.Tensor] = {}
_ERR: dict[int, torch.Tensor] = {}
_HOST_PTR: dict[int, int] = {}


def workspace(device: torch.device, nbytes: int) -> torch.Tensor:
    """Grow-only scratch buffer (256-byte aligned) for split partials."""
    idx = device.index if device.index is not None else torch.cuda.current_device()
    buf = _WS.get(idx)
    if buf is None or buf.numel() < nbytes:
        cap = max(nbytes, 1 << 20, 2 * (buf.numel() if buf is not None else 0))
        buf = torch.empty(cap, dtype=torch.uint8, device=torch.device("cuda", idx))
        _WS[idx] = buf
    return buf


def error_word(device: torch.device) -> torch.Tensor:
    """The int32 device error word the kernels on `device` report into."""
    idx = device.index if device.index is not None else torch.cuda.current_device()
    w = _ERR.get(idx)
    if w is None:
        w = torch.zeros(1, dtype=torch.int32, device=torch.device("cuda", idx))
        _ERR[idx] = w
    return w


def check_device_errors(device: torch.device | None = None) -> None:
    """Synchronise and raise RuntimeError if a kernel on `device` flagged an
    error since the last check (the word is cleared)."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else device
    w = error_word(dev)
    val = ctypes.c_int32(0)
    nat.check(nat.load().fd_read_error(w.data_ptr(), ctypes.byref(val), 1, _stream(dev)), "fd_read_error")
    if val.value != 0:
        raise RuntimeError(f"fastdecode_b200 device error {val.value}: {nat.device_error_string(val.value)}")


def host_device_pointer(t: torch.Tensor) -> int:
    """Device address of t.data_ptr() for a pinned, mapped host tensor (the
    storage base is translated once and cached; views keep their offset)."""
    _check(t.device.type == "cpu", "expected a host tensor")
    _check(t.is_pinned(), "host KV tier must be pinned (pin_memory=True) to be read by the GPU")
    base = t.untyped_storage().data_ptr()
    if base not in _HOST_PTR:
        out = ctypes.c_void_p()
        nat.check(nat.load().fd_host_device_pointer(base, ctypes.byref(out)), "fd_host_device_pointer")
        _HOST_PTR[base] = out.value or 0
    return _HOST_PTR[base] + (t.data_ptr() - base)


def forget_host_pointer(t: torch.Tensor) -> None:
    """Drop the cached device address of t's storage (its memory is about to
    be unregistered)."""
    _HOST_PTR.pop(t.untyped_storage().data_ptr(), None)


# ------------------------------------------------------------- KV tiers


@dataclass
class KVTier:
    """One KV tier viewed as K/V tensors of logical shape [B, KVH, BS, D]
    (any strides with a contiguous last dim).  Device tensors are streamed
    with TMA; pinned host tensors are read over PCIe through their mapped
    device address."""

    k: torch.Tensor
    v: torch.Tensor

    def __post_init__(self) -> None:
        _check(self.k.dim() == 4 and self.v.dim() == 4, "KV tier views must be 4-D [B, KVH, BS, D]")
        _check(self.k.shape == self.v.shape, "K and V views must have the same shape")
        _check(self.k.stride() == self.v.stride(), "K and V views must have the same strides")
        _check(self.k.stride(3) == 1, "head_size must be the contiguous dimension")
        _check(self.k.dtype == self.v.dtype, "K and V dtypes differ")

    @property
    def host(self) -> bool:
        return self.k.device.type == "cpu"

    def to_c(self) -> nat.FdKvTier:
        t = nat.FdKvTier()
        if self.host:
            t.k = host_device_pointer(self.k)
            t.v = host_device_pointer(self.v)
        else:
            t.k = self.k.data_ptr()
            t.v = self.v.data_ptr()
        s = self.k.stride()
        t.blk_stride, t.head_stride, t.tok_stride = s[0], s[1], s[2]
        t.num_blocks = self.k.shape[0]
        t.host_mapped = 1 if self.host else 0
        return t


def _empty_tier() -> nat.FdKvTier:
    return nat.FdKvTier()


def _tier_device(t: KVTier | None) -> torch.device | None:
    if t is None or t.host:
        return None
    return t.k.device


# ------------------------------------------------------------- host-tier staging

_STAGE: dict[int, torch.Tensor] = {}


def stage_host_blocks(tier: KVTier, lo: int, hi: int, device: torch.device) -> KVTier:
    """Copy host-tier blocks [lo, hi) into device memory with the copy engine
    (two cudaMemcpyAsync on the current stream: K, then V) and return the
    device tier over the copy.  The copy engine reads pinned memory faster
    than SM loads over PCIe (B200: 55.6 vs ~51 GB/s), so a step that reads
    most of a compact range of host blocks gains by staging it; decode with
    tier_split + lo as the split so that host id h maps to staged block
    h - lo.  The staging buffer is shared and grow-only (per device): it
    is overwritten by the next staging call on the same device."""
    _check(tier.host, "stage_host_blocks: the tier must be the pinned host tier")
    _check(0 <= lo <= hi <= tier.k.shape[0], f"stage_host_blocks: range [{lo}, {hi}) outside the tier")
    _check(tier.k.is_contiguous() and tier.v.is_contiguous(), "stage_host_blocks: host tier must be contiguous")
    idx = device.index if device.index is not None else torch.cuda.current_device()
    per = tier.k[0].numel()
    need = 2 * max(1, hi - lo) * per
    buf = _STAGE.get(idx)
    if buf is None or buf.numel() < need or buf.dtype != tier.k.dtype:
        buf = torch.empty(need, dtype=tier.k.dtype, device=torch.device("cuda", idx))
        _STAGE[idx] = buf
    shape = (max(1, hi - lo),) + tuple(tier.k.shape[1:])
    k = buf[: need // 2].view(shape)
    v = buf[need // 2: need].view(shape)
    if hi > lo:
        k[: hi - lo].copy_(tier.k[lo:hi], non_blocking=True)
        v[: hi - lo].copy_(tier.v[lo:hi], non_blocking=True)
    return KVTier(k[: max(1, hi - lo)], v[: max(1, hi - lo)])


def host_block_range(block_table: torch.Tensor, lens: torch.Tensor, block_size: int, tier_split: int) -> tuple[int, int]:
    """[lo, hi) of the host-tier blocks (ids >= tier_split, host-relative)
    a step reads, from CPU copies of its block table and lengths."""
    W = block_table.shape[1]
    nb = ((lens.to(torch.int64) + block_size - 1) // block_size).clamp(max=W)
    used = torch.arange(W).unsqueeze(0) < nb.unsqueeze(1)
    ids = block_table.to(torch.int64)[used]
    ids = ids[ids >= tier_split]
    if ids.numel() == 0:
        return 0, 0
    return int(ids.min()) - tier_split, int(ids.max()) - tier_split + 1


@dataclass
class ChunkedStaging:
    """One step's host-tier blocks cut into chunks that are staged into HBM
    one after another on a side stream (plan_chunked_staging).  Part 0 is
    every row's HBM-tier blocks; part j (1..k) is every row's host blocks
    with host-relative ids in chunks[j - 1] = [c_lo, c_hi).  Per part,
    `tables[p]` (int32 [n, W_p], CPU) lists a row's blocks of that part in
    table order, the row's last (partly filled) block moved to the end, with
    ids as the part's decode reads them (HBM ids for part 0, ids relative to
    the staged range [lo, hi) for the others), and `lens[p]` (int32 [n]) is
    the tokens they hold (0: the row has no block in the part)."""

    lo: int
    hi: int
    chunks: list[tuple[int, int]]
    tables: list[torch.Tensor]
    lens: list[torch.Tensor]
    _dev: dict | None = None

    def on(self, device: torch.device) -> list[tuple[torch.Tensor, torch.Tensor]]:
        """(table, lens) of every part on `device`, copied once (one packed
        host-to-device copy) and cached, so that a step captured in a CUDA
        graph copies nothing."""
        key = str(device)
        if self._dev is None:
            self._dev = {}
        if key not in self._dev:
            flat = torch.cat([t.flatten() for t in self.tables] + list(self.lens)).to(device)
            out, o = [], 0
            for t in self.tables:
                out.append(flat[o:o + t.numel()].view(t.shape))
                o += t.numel()
            lens = []
            for ln in self.lens:
                lens.append(flat[o:o + ln.numel()])
                o += ln.numel()
            self._dev[key] = list(zip(out, lens))
        return self._dev[key]


def plan_chunked_staging(block_table: torch.Tensor, lens: torch.Tensor, block_size: int, tier_split: int,
                         chunks: int) -> ChunkedStaging:
    """Cut a step's host-tier range [lo, hi) into `chunks` equal block ranges
    and build the per-part block tables of ChunkedStaging from CPU copies of
    the step's block table and lengths (blocks may lie anywhere in the range:
    each part holds whichever of a row's blocks fall into it)."""
    _check(chunks >= 1, "plan_chunked_staging: chunks must be >= 1")
    n, W = block_table.shape
    BS = block_size
    L = lens.to(torch.int64).clamp(min=0)
    nb = ((L + BS - 1) // BS).clamp(max=W)
    col = torch.arange(W).unsqueeze(0).expand(n, W)
    used = col < nb.unsqueeze(1)
    ids = block_table.to(torch.int64)
    host = used & (ids >= tier_split)
    rel = ids - tier_split
    if bool(host.any()):
        lo, hi = int(rel[host].min()), int(rel[host].max()) + 1
    else:
        lo = hi = 0
    k = max(1, min(chunks, hi - lo)) if hi > lo else 0
    bounds = [lo + ((hi - lo) * j) // k for j in range(k + 1)] if k else []
    spans = [(bounds[j], bounds[j + 1]) for j in range(k)]
    last = col == (nb - 1).unsqueeze(1)  # the row's last block (L - (nb-1)*BS tokens)
    tail = (L - (nb - 1).clamp(min=0) * BS).unsqueeze(1).expand(n, W)
    tok = torch.where(last, tail, torch.full_like(tail, BS))
    masks = [used & (ids < tier_split)] + [host & (rel >= c_lo) & (rel < c_hi) for c_lo, c_hi in spans]
    tables, part_lens = [], []
    for p, m in enumerate(masks):
        key = torch.where(m, torch.where(last, torch.full_like(col, W), col), torch.full_like(col, 2 * W))
        order = key.argsort(dim=1, stable=True)
        cnt = m.sum(dim=1)
        wp = max(1, int(cnt.max()) if n else 1)
        vals = (ids if p == 0 else rel - lo).gather(1, order)[:, :wp]
        keep = torch.arange(wp).unsqueeze(0) < cnt.unsqueeze(1)
        tables.append(torch.where(keep, vals, torch.zeros_like(vals)).to(torch.int32).contiguous())
        part_lens.append(torch.where(m, tok, torch.zeros_like(tok)).sum(dim=1).to(torch.int32))
    return ChunkedStaging(lo, hi, spans, tables, part_lens)


_SIDE: dict[int, torch.cuda.Stream] = {}
_PARTS: dict[int, torch.Tensor] = {}


def _side_stream(device: torch.device) -> torch.cuda.Stream:
    idx = device.index if device.index is not None else torch.cuda.current_device()
    st = _SIDE.get(idx)
    if st is None:
        st = torch.cuda.Stream(torch.device("cuda", idx))
        _SIDE[idx] = st
    return st


def decode_staged_chunks(q: torch.Tensor, tiers: tuple[KVTier | None, KVTier | None],
                         scale: float, out: torch.Tensor, lse: torch.Tensor | None, plan: ChunkedStaging, *,
                         q_rows: torch.Tensor | None = None, out_rows: torch.Tensor | None = None,
                         parts_buf: torch.Tensor | None = None) -> None:
    """Decode over an HBM tier and a pinned host tier whose blocks are
    staged into HBM chunk by chunk, the copies overlapping the decode.

    The copy engine copies chunk j of `plan` into the staging buffer on a
    side stream and records an event; on the current stream the HBM-tier
    blocks are decoded first (while the first chunk copies), then each
    chunk's blocks once its event has fired, every part into fp32 partials
    (o, lse), and one P-way log-sum-exp merge (fd_merge_partials) combines
    the k + 1 partials into `out` (rows out_rows[i] or i) and `lse` [H, n].
    Only the last chunk's decode and the merge follow the last copy.  The
    staging buffer is the one stage_host_blocks uses; the side stream waits
    for earlier work on the current stream before overwriting it.  The
    side stream forks from and joins the current stream, so a step can be
    captured in a CUDA graph (`parts_buf`: fp32 partials owned by the
    caller, e.g. for a captured step)."""
    host = tiers[1]
    _check(host is not None and host.host, "decode_staged_chunks: tiers[1] must be the pinned host tier")
    _check(host.k.is_contiguous() and host.v.is_contiguous(), "decode_staged_chunks: host tier must be contiguous")
    dev = q.device
    idx = dev.index if dev.index is not None else torch.cuda.current_device()
    n = plan.tables[0].shape[0]
    H, D = q.shape[-2], q.shape[-1]
    P = 1 + len(plan.chunks)
    stride = n * H * D + H * n
    if parts_buf is None:
        parts_buf = _PARTS.get(idx)
        if parts_buf is None or parts_buf.numel() < P * stride:
            parts_buf = torch.empty(P * stride, dtype=torch.float32, device=dev)
            _PARTS[idx] = parts_buf
    _check(parts_buf.dtype == torch.float32 and parts_buf.numel() >= P * stride, "parts_buf too small")
    parts = parts_buf[: P * stride].view(P, stride)
    main = torch.cuda.current_stream(dev)
    side = _side_stream(dev)
    lo, hi = plan.lo, plan.hi
    per = host.k[0].numel()
    need = 2 * max(1, hi - lo) * per
    buf = _STAGE.get(idx)
    if buf is None or buf.numel() < need or buf.dtype != host.k.dtype:
        buf = torch.empty(need, dtype=host.k.dtype, device=torch.device("cuda", idx))
        _STAGE[idx] = buf
    shape = (max(1, hi - lo),) + tuple(host.k.shape[1:])
    kb = buf[: need // 2].view(shape)
    vb = buf[need // 2: need].view(shape)
    staged = KVTier(kb, vb)
    dev_parts = plan.on(dev)

    def part(p: int, t: tuple[KVTier | None, KVTier | None], split: int) -> None:
        bt, ln = dev_parts[p]
        o = parts[p, : n * H * D].view(n, H, D)
        ls = parts[p, n * H * D:].view(H, n)
        a = decode_args(q, t, split, bt, ln, scale, o, ls, q_rows=q_rows,
                        max_len=int(plan.lens[p].max()) if n else 0)
        launch_decode(a, dev)

    ready = torch.cuda.Event()
    ready.record(main)  # earlier readers of the staging buffer come first
    side.wait_event(ready)
    evs = []
    with torch.cuda.stream(side):
        for c_lo, c_hi in plan.chunks:
            kb[c_lo - lo: c_hi - lo].copy_(host.k[c_lo:c_hi], non_blocking=True)
            vb[c_lo - lo: c_hi - lo].copy_(host.v[c_lo:c_hi], non_blocking=True)
            ev = torch.cuda.Event()
            ev.record(side)
            evs.append(ev)
    # no record_stream for the side stream: every use of the buffer there is
    # followed, on the current stream, by a wait on its event, so the
    # buffer's lifetime on the current stream covers the side stream's too
    if tiers[0] is not None:
        part(0, (tiers[0], None), 1 << 40)
    else:
        parts[0, : n * H * D].zero_()
        parts[0, n * H * D:].fill_(float("-inf"))
    for j, ev in enumerate(evs):
        main.wait_event(ev)
        part(j + 1, (None, staged), 0)
    if out_rows is None:
        merge_partials(parts, P, n, H, D, out, lse)
    else:
        tmp = torch.empty(n, H, D, dtype=out.dtype, device=dev)
        merge_partials(parts, P, n, H, D, tmp, lse)
        out.index_copy_(0, out_rows.to(torch.int64), tmp)


# ------------------------------------------------------------- decode


def choose_tiles_per_split(total_tokens: int, n_ctas_per_row: int, block_size: int,
                           num_sms: int = 148) -> int:
    """Tiles (min(block_size,16) tokens) per split so that the grid holds about
    eight waves of two CTAs per SM, given the real token count of the batch."""
    tt = block_size if block_size <= 16 else 16
    tiles = max(1, math.ceil(total_tokens / tt)) * max(1, n_ctas_per_row)
    tps = max(8, math.ceil(tiles / (num_sms * 2 * 8)))
    return (tps + 3) // 4 * 4


def decode_kernel_name(dtype: torch.dtype, head_size: int, num_heads: int, num_kv_heads: int, block_size: int,
                       n: int, tiles_per_split: int = 0) -> str:
    """Name of the kernel fd_decode_attn launches for this shape, mirroring
    the library's dispatch (fd_decode.cu geometry(), fd_decode_mma.cu
    mma_eligible()): the tcgen05 kernel for 16-bit KV, head size 128, query
    group 2/4/8, block size a multiple of 16 and the persistent schedule
    (<= 1024 rows, no explicit split), unless FASTDECODE_B200_MMA=0."""
    G = num_heads // max(1, num_kv_heads)
    persistent = tiles_per_split <= 0 and 0 < n <= 1024
    mma = (persistent and dtype in (torch.float16, torch.bfloat16) and head_size == 128 and G in (2, 4, 8)
           and block_size % 16 == 0 and not os.environ.get("FASTDECODE_B200_MMA", "").startswith("0"))
    return "fd_decode_mma_kernel" if mma else "fd_decode_kernel"


def decode_args(q: torch.Tensor, tiers: tuple[KVTier | None, KVTier | None], tier_split: int,
                block_table: torch.Tensor, lens: torch.Tensor, scale: float, out: torch.Tensor,
                lse: torch.Tensor | None = None, *, q_rows: torch.Tensor | None = None,
                out_rows: torch.Tensor | None = None, max_len: int = 0,
                tiles_per_split: int = 0, n: int | None = None,
                bt_rows: torch.Tensor | None = None,
                workspace_buf: torch.Tensor | None = None, pdl: bool = False) -> nat.FdDecodeArgs:
    """Validate and pack the arguments of fd_decode_attn (workspace included).
    The tensors must stay alive, unmoved, while the returned args are used.
    With bt_rows (int32 [n]) work row i reads table row bt_rows[i]; a
    negative out_rows[i] writes nothing for row i (a device-built decode
    list, plan.plan_on_device).  workspace_buf (uint8, on q's device) replaces
    the shared grow-only workspace, e.g. for launches captured in a CUDA graph,
    whose pointers must stay valid for the graph's lifetime.  pdl=True
    launches the decode as a programmatic dependent of the kernel ahead on
    the stream (FD_DECODE_PDL): only when that kernel writes none of lens,
    block_table, the row maps and q (e.g. it is the layer's KV write or the
    previous decode's combine)."""
    lib = nat.load()
    dev = q.device
    _check(dev.type == "cuda", "q must be a CUDA tensor")
    H, D = q.shape[-2], q.shape[-1]
    _check(q.stride(-1) == 1 and out.stride(-1) == 1, "q and out need a contiguous head dim")
    n = (block_table.shape[0] if bt_rows is None else bt_rows.shape[0]) if n is None else n
    if bt_rows is not None:
        _check(bt_rows.dtype == torch.int32 and bt_rows.device == dev and bt_rows.numel() >= n,
               "bt_rows must be int32 on q's device with n entries")
    for nm, rows in (("q_rows", q_rows), ("out_rows", out_rows)):
        if rows is not None:  # the kernels read them as int64 (fd_decode_args)
            _check(rows.dtype == torch.int64 and rows.device == dev and rows.is_contiguous() and rows.numel() >= n,
                   f"{nm} must be a contiguous int64 tensor on q's device with n entries")
    _check(block_table.dtype == torch.int32 and lens.dtype == torch.int32, "block_table and lens must be int32")
    _check(block_table.stride(-1) == 1, "block_table rows must be contiguous")
    _check(block_table.device == dev and lens.device == dev, "block_table and lens must be on q's device")
    t0, t1 = tiers
    ref = t0 if t0 is not None else t1
    _check(ref is not None, "at least one KV tier is required")
    _check(ref.k.dtype == q.dtype, "q and KV cache dtypes differ")
    KVH, BS = ref.k.shape[1], ref.k.shape[2]
    _check(ref.k.shape[3] == D, "head size mismatch")
    for t in tiers:
        if t is not None:
            _check(t.k.shape[1:] == ref.k.shape[1:], "tiers must share [KVH, BS, D]")
            _check(t.host or t.k.device == dev, "device tier must live on q's device")
    a = nat.FdDecodeArgs()
    a.q = q.data_ptr()
    a.q_stride_n = q.stride(0)
    a.q_stride_h = q.stride(1)
    a.q_rows = _ptr(q_rows)
    a.tier[0] = t0.to_c() if t0 is not None else _empty_tier()
    a.tier[1] = t1.to_c() if t1 is not None else _empty_tier()
    a.tier_split = int(tier_split)
    a.block_table = block_table.data_ptr()
    a.bt_stride = block_table.stride(0)
    a.bt_width = block_table.shape[1]
    a.lens = lens.data_ptr()
    a.n = n
    a.num_heads = H
    a.num_kv_heads = KVH
    a.head_size = D
    a.block_size = BS
    a.scale = float(scale)
    a.dtype = dtype_code(q.dtype)
    a.out = out.data_ptr()
    a.out_dtype = dtype_code(out.dtype)
    a.out_stride_n = out.stride(0)
    a.out_stride_h = out.stride(1)
    a.out_rows = _ptr(out_rows)
    if lse is not None:
        _check(lse.dtype == torch.float32 and lse.device == dev, "lse must be fp32 on q's device")
        a.lse = lse.data_ptr()
        a.lse_stride_h = lse.stride(0)
        a.lse_stride_n = lse.stride(1)
    a.bt_rows = _ptr(bt_rows)
    a.flags = nat.FD_DECODE_PDL if pdl else 0
    a.max_len = int(max_len)
    a.tiles_per_split = int(tiles_per_split)
    a.error = error_word(dev).data_ptr()
    need = lib.fd_decode_workspace_size(ctypes.byref(a))
    if need:
        if workspace_buf is not None:
            _check(workspace_buf.device == dev and workspace_buf.dtype == torch.uint8 and workspace_buf.numel() >= need,
                   f"workspace_buf must be uint8 on q's device with >= {need} bytes")
            ws = workspace_buf
        else:
            ws = workspace(dev, need)
        a.workspace = ws.data_ptr()
        a.workspace_bytes = ws.numel()
    return a


def launch_decode(a: nat.FdDecodeArgs, device: torch.device, phase: str = "all") -> None:
    """Launch fd_decode_attn ("all") or one of its two kernels ("partials",
    "combine") on the current stream of `device`."""
    lib = nat.load()
    fn = {"all": lib.fd_decode_attn, "partials": lib.fd_decode_attn_partials,
          "combine": lib.fd_decode_attn_combine}[phase]
    nat.check(fn(ctypes.byref(a), _stream(device)), f"fd_decode_attn[{phase}]")


def decode_tiered(q: torch.Tensor, tiers: tuple[KVTier | None, KVTier | None], tier_split: int,
                  block_table: torch.Tensor, lens: torch.Tensor, scale: float, out: torch.Tensor,
                  lse: torch.Tensor | None = None, **kw) -> None:
    """Paged decode attention over a two-tier block table (fd_decode_attn).

    q [T, H, D] (rows q_rows[i] or i), tiers[0]/tiers[1] the HBM and host
    tiers (ids < tier_split and >= tier_split), block_table [n, W] int32,
    lens [n] int32, out [*, H, D] (rows out_rows[i] or i; q dtype or fp32),
    lse [H, n] fp32 or None.  Keywords: q_rows, out_rows, max_len,
    tiles_per_split, n (see decode_args), and host_range = (lo, hi): stage
    host-tier blocks [lo, hi) (every host block the step reads) into device
    memory with the copy engine first (stage_host_blocks) and decode from
    there."""
    host_range = kw.pop("host_range", None)
    if host_range is not None and tiers[1] is not None and tiers[1].host:
        lo, hi = host_range
        tiers = (tiers[0], stage_host_blocks(tiers[1], lo, hi, q.device))
        tier_split = tier_split + lo
    a = decode_args(q, tiers, tier_split, block_table, lens, scale, out, lse, **kw)
    launch_decode(a, q.device)


def decode_attn(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                block_table: torch.Tensor, lens: torch.Tensor, scale: float,
                out: torch.Tensor, lse: torch.Tensor) -> None:
    """Reference signature (fastdecode/csrc/cpu_attn.cpp:456-489).

    q [n,H,D] on the GPU; k_cache/v_cache [C,KVH,BS,D] contiguous, either on
    the GPU or pinned host memory (the host tier, read over PCIe);
    block_table [n,W] int32 cache-relative ids; lens [n] int32; out [n,H,D]
    (q dtype); lse [H,n] fp32."""
    for t, name in ((q, "q"), (k_cache, "k_cache"), (v_cache, "v_cache"), (block_table, "block_table"),
                    (lens, "lens"), (out, "out"), (lse, "lse")):
        _check(t.is_contiguous(), f"{name} must be contiguous")
    _check(q.dim() == 3 and k_cache.dim() == 4 and v_cache.shape == k_cache.shape,
           "expected q [n,H,D] and caches [C,KVH,BS,D]")
    _check(block_table.dtype == torch.int32 and lens.dtype == torch.int32, "block_table and lens must be int32")
    _check(lse.dtype == torch.float32, "lse must be float32")
    _check(q.dtype == k_cache.dtype and out.dtype == q.dtype, "q, cache and out dtypes must match")
    n, H, D = q.shape
    KVH, BS = k_cache.shape[1], k_cache.shape[2]
    _check(k_cache.shape[3] == D, "head size mismatch")
    _check(H % KVH == 0, "num_heads must be a multiple of num_kv_heads")
    _check(block_table.dim() == 2 and block_table.shape[0] == n and lens.shape[0] == n,
           "block_table [n, W] and lens [n] expected")
    _check(out.shape == q.shape and lse.shape == (H, n), "out [n,H,D] and lse [H,n] expected")
    if n == 0:
        return
    _check(q.is_cuda, "q must be a CUDA tensor")
    dev = q.device
    bt = block_table if block_table.device == dev else block_table.to(dev, non_blocking=True)
    ln = lens if lens.device == dev else lens.to(dev, non_blocking=True)
    decode_tiered(q, (KVTier(k_cache, v_cache), None), 1 << 62, bt, ln, scale, out, lse)


# ------------------------------------------------------------- KV write


def store_kv_tiered(key: torch.Tensor, value: torch.Tensor, slots: torch.Tensor,
                    tiers: tuple[KVTier | None, KVTier | None], tier_split_blocks: int) -> None:
    """Write new K/V rows [m, KVH, D] to slots (int64, -1 = skip) in either tier."""
    lib = nat.load()
    dev = key.device
    _check(dev.type == "cuda", "key must be a CUDA tensor")
    _check(slots.dtype == torch.int64 and slots.device == dev, "slots must be int64 on key's device")
    _check(key.stride(-1) == 1 and value.stride(-1) == 1, "key/value need a contiguous head dim")
    t0, t1 = tiers
    ref = t0 if t0 is not None else t1
    _check(ref is not None and key.dtype == ref.k.dtype and value.dtype == key.dtype, "dtype mismatch")
    m = slots.shape[0]
    KVH, BS, D = ref.k.shape[1], ref.k.shape[2], ref.k.shape[3]
    _check(key.shape[1] == KVH and key.shape[2] == D and value.shape[1:] == key.shape[1:],
           "key/value must be [m, KVH, D]")
    arr = (nat.FdKvTier * 2)()
    arr[0] = t0.to_c() if t0 is not None else _empty_tier()
    arr[1] = t1.to_c() if t1 is not None else _empty_tier()
    nat.check(lib.fd_store_kv(key.data_ptr(), key.stride(0), key.stride(1), value.data_ptr(),
                              value.stride(0), value.stride(1), slots.data_ptr(), m, KVH, D, BS,
                              dtype_code(key.dtype), arr, int(tier_split_blocks),
                              error_word(dev).data_ptr(), _stream(dev)), "fd_store_kv")


def store_kv(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, k_cache: torch.Tensor,
             v_cache: torch.Tensor) -> None:
    """Reference signature (fastdecode/csrc/cpu_attn.cpp:492-517): k, v [m,KVH,D]
    on the GPU; slots [m] int64 cache-relative; caches [C,KVH,BS,D] on the GPU
    or pinned host memory.  An out-of-range slot raises RuntimeError and
    nothing is written."""
    for t, name in ((k, "k"), (v, "v"), (slots, "slots"), (k_cache, "k_cache"), (v_cache, "v_cache")):
        _check(t.is_contiguous(), f"{name} must be contiguous")
    _check(slots.dtype == torch.int64, "slots must be int64")
    _check(k.dtype == k_cache.dtype and v.dtype == k.dtype, "dtype mismatch")
    m = k.shape[0]
    if m == 0:
        return
    C, KVH, BS, D = k_cache.shape
    _check(k.shape[1] == KVH and k.shape[2] == D and v.shape == k.shape, "k/v must be [m, KVH, D]")
    cap = C * BS
    if slots.device.type == "cpu":
        bad = (slots < 0) | (slots >= cap)
        if bool(bad.any()):
            raise RuntimeError(f"CPU slot out of range: {int(slots[bad][0])}")
        slots = slots.to(k.device, non_blocking=True)
    dev = k.device
    store_kv_tiered(k, v, slots, (KVTier(k_cache, v_cache), None), 1 << 62)
    if not torch.cuda.is_current_stream_capturing():
        try:
            check_device_errors(dev)
        except RuntimeError as e:
            raise RuntimeError(f"CPU slot out of range ({e})") from None


# ------------------------------------------------------------- prefill


def prefill_attn(q: torch.Tensor, out: torch.Tensor, q_start: torch.Tensor, q_len: torch.Tensor,
                 k_len: torch.Tensor, scale: float, *, kv: KVTier | None = None,
                 block_table: torch.Tensor | None = None, bt_row: torch.Tensor | None = None,
                 k: torch.Tensor | None = None, v: torch.Tensor | None = None,
                 total_q: int | None = None) -> None:
    """Causal prefill attention on the tensor cores (fd_prefill_attn), the
    replacement of flash_attn_varlen_func(causal=True) for the P and F
    classes (fastdecode/backend.py:317-340).

    q, out [T, H, 128] fp16/bf16 (batch rows); per request r (int32 device
    tensors [n]): q_start (first query row), q_len, k_len >= q_len; query i
    sees keys 0 .. k_len - q_len + i.  Keys/values either from the paged
    HBM tier (kv [B, KVH, BS, D] views, block_table [R, W] int32, optional
    bt_row [n] int32 table row of each request) or from the batch's own new
    rows (k, v [T, KVH, D]; key j of request r is row q_start[r] + j).
    total_q bounds the grid (sum of q_len; computed with a host sync when
    not given).  Only the requests' rows of out are written."""
    lib = nat.load()
    dev = q.device
    _check(dev.type == "cuda", "q must be a CUDA tensor")
    _check(q.dim() == 3 and out.shape == q.shape and out.dtype == q.dtype, "q and out must be [T, H, D] alike")
    _check(q.stride(-1) == 1 and out.stride(-1) == 1, "q and out need a contiguous head dim")
    for nm, t in (("q_start", q_start), ("q_len", q_len), ("k_len", k_len)) + ((("bt_row", bt_row),) if bt_row is not None else ()):
        _check(t.dtype == torch.int32 and t.device == dev and t.is_contiguous(), f"{nm} must be contiguous int32 on q's device")
    n = q_len.numel()
    _check(q_start.numel() == n and k_len.numel() == n and (bt_row is None or bt_row.numel() == n),
           "per-request arrays must have the same length")
    T, H, D = q.shape
    a = nat.FdPrefillArgs()
    a.q, a.q_stride_t, a.q_stride_h = q.data_ptr(), q.stride(0), q.stride(1)
    a.out, a.out_stride_t, a.out_stride_h = out.data_ptr(), out.stride(0), out.stride(1)
    t = nat.FdKvTier()
    if block_table is not None:
        _check(kv is not None and not kv.host, "paged prefill needs the device KV tier")
        _check(block_table.dtype == torch.int32 and block_table.device == dev and block_table.stride(-1) == 1,
               "block_table must be int32 on q's device with contiguous rows")
        _check(kv.k.dtype == q.dtype and kv.k.shape[3] == D, "KV tier dtype / head size mismatch")
        t = kv.to_c()
        KVH, BS = kv.k.shape[1], kv.k.shape[2]
        a.block_table, a.bt_stride, a.bt_width = block_table.data_ptr(), block_table.stride(0), block_table.shape[1]
        a.block_size = BS
    else:
        _check(k is not None and v is not None, "give either kv + block_table or k and v")
        _check(k.shape == v.shape and k.stride() == v.stride() and k.dim() == 3 and k.stride(-1) == 1,
               "k and v must be [T, KVH, D] alike with a contiguous head dim")
        _check(k.dtype == q.dtype and k.device == dev and k.shape[2] == D, "k / v dtype, device or head size mismatch")
        KVH = k.shape[1]
        t.k, t.v = k.data_ptr(), v.data_ptr()
        t.blk_stride, t.head_stride, t.tok_stride = 0, k.stride(1), k.stride(0)
        t.num_blocks = k.shape[0]
        a.block_size = 0
    a.kv = t
    a.num_tokens = T
    a.q_start, a.q_len, a.k_len = q_start.data_ptr(), q_len.data_ptr(), k_len.data_ptr()
    a.bt_row = _ptr(bt_row)
    a.n, a.num_heads, a.num_kv_heads, a.head_size = n, H, KVH, D
    a.scale = float(scale)
    a.dtype = dtype_code(q.dtype)
    a.total_q = int(q_len.sum().item()) if total_q is None else int(total_q)
    a.error = error_word(dev).data_ptr()
    nat.check(lib.fd_prefill_attn(ctypes.byref(a), _stream(dev)), "fd_prefill_attn")


# ------------------------------------------------------------- multi-token steps
#
# These calls pack their C struct in one struct.pack (a ctypes field store each
# would cost more than the launch) and read each tensor's metadata once, since a
# decode step's call is bound by this code; they run on the device of their
# tensors whatever the current one is, and take their workspace from torch's
# caching allocator per call: it belongs to the current stream, and to the
# graph when one is being captured, so calls on other streams and other graphs
# never share it.

_TIER_FMT = "PPqqqqii"
_ATTN_STRUCT = struct.Struct("@PqqPqqPqq" + 2 * _TIER_FMT + "qPqPPPPPiiiiiiifiiiiPNP")
_ROPE_STRUCT = struct.Struct("@" + 5 * "Pqq" + "PqPqP" + 2 * _TIER_FMT + f"q9i{nat.ROPE_MAX_PAIRS}siP")
_TABLES_STRUCT = struct.Struct("@PPPqiiPPiiPPqqiiPPPPPPPP")
_TRIM_STRUCT = struct.Struct("@PPPPPqiiPPiiPPqqiiPP")
_VERIFY_STRUCT = struct.Struct("@PqPqqPqPPPqPPPPPiiiiiiP")
_KEY_WEIGHTS_STRUCT = struct.Struct(_ATTN_STRUCT.format + "PPqP")
_SELECT_STRUCT = struct.Struct("@PPqPqPPPPPPiiiiiiiiP")
_MOVE_STRUCT = struct.Struct("@PPP" + 2 * _TIER_FMT + "qPqPPqiiiiiiiiP")
_NO_TIER = (0, 0, 0, 0, 0, 0, 0, 0)


def _launch(fn, packed: bytes, idx: int, what: str) -> None:
    """Call a C entry point on the current stream of device `idx`."""
    if idx != torch._C._cuda_getDevice():
        with torch.cuda.device(idx):
            status = fn(packed, torch._C._cuda_getCurrentRawStream(idx))
    else:
        status = fn(packed, torch._C._cuda_getCurrentRawStream(idx))
    if status:
        nat.check(status, what)


def _error_ptr(idx: int) -> int:
    w = _ERR.get(idx)
    return (w if w is not None else error_word(torch.device("cuda", idx))).data_ptr()


def _tier_fields(t: KVTier | None, idx: int, dtype: torch.dtype, shape: tuple) -> tuple:
    """The C fields of a tier of [KVH, BS, D] = shape blocks."""
    if t is None:
        return _NO_TIER
    k, v = t.k, t.v
    if k.dtype is not dtype:
        raise RuntimeError("the KV tier's dtype differs")
    sizes = k.shape
    if sizes[1:] != shape:
        raise RuntimeError("the KV tiers must be [blocks, KVH, block_size, D] alike")
    B, s = sizes[0], k.stride()
    if k.get_device() == idx and v.get_device() == idx:
        return (k.data_ptr(), v.data_ptr(), s[0], s[1], s[2], B, 0, 0)
    if k.is_cuda or v.is_cuda:
        raise RuntimeError("a device tier must live on the tensors' device")
    return (host_device_pointer(k), host_device_pointer(v), s[0], s[1], s[2], B, 1, 0)


def _i32(t: torch.Tensor, idx: int, n: int, name: str) -> int:
    if t.dtype is not torch.int32 or t.get_device() != idx or t.numel() < n or not t.is_contiguous():
        raise RuntimeError(f"{name} must be a contiguous int32 tensor of at least {n} entries on the call's device")
    return t.data_ptr()


def _rows3(t: torch.Tensor, idx: int, dtype: torch.dtype, name: str) -> tuple:
    """(pointer, stride 0, stride 1) of a [*, *, D] tensor with contiguous rows."""
    s0, s1, s2 = t.stride()
    if s2 != 1 or t.dtype is not dtype or t.get_device() != idx:
        raise RuntimeError(f"{name} must share q's dtype and device and have a contiguous head dim")
    return t.data_ptr(), s0, s1


def _block_table(t: torch.Tensor) -> tuple[int, int, int]:
    """(device index, R, W) of a block table int32 [R, W]."""
    idx = t.get_device()
    if idx < 0:
        raise RuntimeError("block_table must be a CUDA tensor")
    if t.dtype is not torch.int32 or t.dim() != 2 or (t.stride(1) != 1 and t.shape[1] != 1):
        raise RuntimeError("block_table must be int32 [R, W] with contiguous rows")
    return idx, *t.shape


@dataclass
class FreeBlocks:
    """The free blocks of both tiers as stacks in device memory: hbm / host
    int32 [capacity] (host ids start at num_gpu_blocks; None: no such tier),
    counts int32 [2], the next block to take at counts - 1."""

    hbm: torch.Tensor | None
    host: torch.Tensor | None
    counts: torch.Tensor


def _read_header(header: torch.Tensor, what: str) -> dict[str, int]:
    h = header.tolist()
    flags = h[nat.TABLES_FIELDS["flags"]]
    if flags:
        why = ", ".join(text for bit, text in nat.TABLES_FLAGS.items() if flags & bit)
        raise RuntimeError(f"{what} refused the step: {why}")
    return {k: h[i] for k, i in nat.TABLES_FIELDS.items()}


class StepTables:
    """Device buffers that extend_tables fills for a step of up to R requests
    and T new tokens.  seq_lens and counts may be the caller's own tensors:
    the prior lengths and the free stacks' counts, to step them in place.  A
    call for fewer requests fills the first entries of each and leaves those
    behind as they were."""

    def __init__(self, R: int, T: int, device, seq_lens: torch.Tensor | None = None,
                 counts: torch.Tensor | None = None):
        z = lambda n, dt: torch.zeros(n, dtype=dt, device=device)  # noqa: E731
        self.R, self.T = int(R), int(T)
        self.seq_lens = z(R, torch.int32) if seq_lens is None else seq_lens
        self.counts = z(2, torch.int32) if counts is None else counts
        self.query_lens, self.query_start_loc = z(R, torch.int32), z(R + 1, torch.int32)
        self.slot_mapping, self.positions = z(T, torch.int64), z(T, torch.int64)
        self.header = z(nat.TABLES_HEADER_LEN, torch.int32)

    def read_header(self) -> dict[str, int]:
        """The header by name (synchronises); raises if the step was refused."""
        return _read_header(self.header, "extend_tables")


def extend_tables(new_lens: torch.Tensor, prior_lens: torch.Tensor, block_table: torch.Tensor, free: FreeBlocks,
                  num_gpu_blocks: int, num_cpu_blocks: int, block_size: int,
                  out: StepTables | None = None, max_tokens: int | None = None,
                  evicted: torch.Tensor | None = None) -> StepTables:
    """Block tables, slots and positions of a step from the requests' lengths
    (fd_extend_tables), on the GPU without any host synchronisation.

    new_lens int32 [R]: new tokens of each request (0: none, -1: the request
    ends and gives its blocks back); prior_lens int32 [R]: its tokens in the
    cache; block_table int32 [R, W], changed in place; free: the stacks, HBM
    blocks are taken first.  Fills and returns `out` (or a new StepTables for
    max_tokens new tokens): seq_lens, query_lens, query_start_loc, slot_mapping
    (-1 behind the last token), positions, counts and the header; its seq_lens,
    query_start_loc and slot_mapping are what plan.plan_on_device takes, its
    query_lens (0 where new_lens is -1) and query_start_loc chunk_attn's and
    cross_attn's q_len and q_start.  The next step's prior_lens and free.counts
    are its seq_lens and counts, which may be the same tensors.  A step that
    cannot be applied as a whole changes nothing, has no tokens and sets the
    error word (check_device_errors; StepTables.read_header says why).
    evicted int32 [R]: the tokens that trim_tables cut from each request to
    meet a budget; positions are ahead of cache indices by as many, and an
    ended request's entry becomes 0."""
    idx, R, W = _block_table(block_table)
    if R > 1 and block_table.stride(0) < W:
        raise RuntimeError("block_table's rows must not overlap")
    if out is None:
        _check(max_tokens is not None, "give out or max_tokens")
        out = StepTables(R, max_tokens, block_table.device)
    T = out.T if max_tokens is None else int(max_tokens)
    if out.R < R or out.T < T or out.header.get_device() != idx:
        raise RuntimeError("out is too small for the step, or on another device")
    hbm, host, counts = free.hbm, free.host, free.counts
    packed = _TABLES_STRUCT.pack(
        _i32(new_lens, idx, R, "new_lens"), _i32(prior_lens, idx, R, "prior_lens"), block_table.data_ptr(),
        max(W, block_table.stride(0)), W, R, 0 if hbm is None else _i32(hbm, idx, 0, "free.hbm"),
        0 if host is None else _i32(host, idx, 0, "free.host"), 0 if hbm is None else hbm.numel(),
        0 if host is None else host.numel(), _i32(counts, idx, 2, "free.counts"), _i32(out.counts, idx, 2, "out.counts"),
        num_gpu_blocks, num_cpu_blocks, block_size, T, _i32(out.seq_lens, idx, R, "out.seq_lens"),
        out.query_start_loc.data_ptr(), out.slot_mapping.data_ptr(), out.positions.data_ptr(), out.header.data_ptr(),
        _error_ptr(idx), _i32(out.query_lens, idx, R, "out.query_lens"),
        0 if evicted is None else _i32(evicted, idx, R, "evicted"))
    _launch(nat.load().fd_extend_tables, packed, idx, "fd_extend_tables")
    return out


class _Buffers:
    """int32 buffers of one device, checked when they are made (a call then only
    takes their addresses), so their names are not to be bound again."""

    def __init__(self, device, **buffers):
        made = {k: v if isinstance(v, torch.Tensor) else torch.zeros(v, dtype=torch.int32, device=device)
                for k, (v, _) in buffers.items()}
        idx = next(iter(made.values())).get_device()
        for name, t in made.items():
            need = buffers[name][1]
            if t.dtype is not torch.int32 or t.get_device() != idx or t.numel() < need or not t.is_contiguous():
                raise RuntimeError(f"{name} must be a contiguous int32 tensor of at least {need} entries on one device with the others")
        self.__dict__.update(made, idx=idx)

    def __setattr__(self, name, value):
        raise AttributeError(f"{type(self).__name__}.{name} is not to be bound again: make a new {type(self).__name__}")


class TrimTables(_Buffers):
    """Device buffers that trim_tables fills for up to R requests: the lengths
    after it, the free stacks' counts and the header.  seq_lens and counts may
    be the caller's own tensors, to step them in place."""

    def __init__(self, R: int, device, seq_lens: torch.Tensor | None = None, counts: torch.Tensor | None = None):
        super().__init__(device, seq_lens=(R if seq_lens is None else seq_lens, R), counts=(2 if counts is None else counts, 2),
                         header=(nat.TABLES_HEADER_LEN, nat.TABLES_HEADER_LEN))
        self.__dict__["R"] = int(R)

    def read_header(self) -> dict[str, int]:
        """The header by name (synchronises); raises if the call was refused."""
        return _read_header(self.header, "trim_tables")


def trim_tables(keep_lens: torch.Tensor, seq_lens: torch.Tensor, block_table: torch.Tensor, free: FreeBlocks,
                num_gpu_blocks: int, num_cpu_blocks: int, block_size: int, out: TrimTables | None = None, *,
                evicted: torch.Tensor | None = None, max_cut: int = 0) -> TrimTables:
    """Cut requests to their first keep_lens tokens and push the blocks behind
    them onto their tier's free stack (fd_trim_tables), without any host
    synchronisation: after verify_drafts, whose keep_lens drops the rejected
    drafts, or after every layer's move_keys.

    keep_lens int32 [R]: the tokens that stay (below 0, or not below seq_lens:
    the request is left as it is); seq_lens int32 [R]: its tokens in the cache;
    block_table int32 [R, W], which stays as it is.  Fills and returns `out`:
    seq_lens, counts and the header (freed_hbm, freed_host, max_seq); they may
    be the call's own seq_lens and free.counts.  evicted int32 [R] (cuts to a
    budget only) grows by what each request lost.  max_cut: the host's bound on
    that, if it knows one.  A call that cannot be applied as a whole changes
    nothing and sets the error word (check_device_errors;
    TrimTables.read_header says why)."""
    idx, R, W = _block_table(block_table)
    if out is None:
        out = TrimTables(R, block_table.device)
    if out.R < R or out.idx != idx:
        raise RuntimeError("out is too small, or on another device")
    hbm, host, counts = free.hbm, free.host, free.counts
    packed = _TRIM_STRUCT.pack(
        _i32(keep_lens, idx, R, "keep_lens"), _i32(seq_lens, idx, R, "seq_lens"), out.seq_lens.data_ptr(),
        0 if evicted is None else _i32(evicted, idx, R, "evicted"), block_table.data_ptr(), block_table.stride(0), W, R,
        0 if hbm is None else _i32(hbm, idx, 0, "free.hbm"), 0 if host is None else _i32(host, idx, 0, "free.host"),
        0 if hbm is None else hbm.numel(), 0 if host is None else host.numel(), _i32(counts, idx, 2, "free.counts"),
        out.counts.data_ptr(), num_gpu_blocks, num_cpu_blocks, block_size, max_cut, out.header.data_ptr(),
        _error_ptr(idx))
    _launch(nat.load().fd_trim_tables, packed, idx, "fd_trim_tables")
    return out


@lru_cache(maxsize=64)
def rope_axes(sections: tuple[int, ...], turns: bool = False) -> bytes:
    """The axis of each rotated pair.  sections[a] pairs belong to axis a: in
    blocks (axis 0's pairs first), or, with turns, dealt out one after the
    other, an axis that has all its pairs being passed over."""
    _check(1 <= len(sections) <= nat.ROPE_MAX_AXES and all(n >= 0 for n in sections) and sum(sections) > 0,
           f"sections: the pairs of 1 to {nat.ROPE_MAX_AXES} axes")
    _check(sum(sections) <= nat.ROPE_MAX_PAIRS, f"at most {nat.ROPE_MAX_PAIRS} rotated pairs")
    if not turns:
        return bytes(a for a, n in enumerate(sections) for _ in range(n))
    order: list[int] = []
    for i in range(max(sections)):
        order += [a for a, n in enumerate(sections) if i < n]
    return bytes(order)


def rope_store_kv(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor,
                  slots: torch.Tensor | None, tiers: tuple[KVTier | None, KVTier | None], tier_split: int, *,
                  sections: tuple[int, ...] | None = None, turns: bool = False, pairs: bool = False,
                  q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotate q and k by multi-axis positions and write the rotated k, and v,
    to their cache slots in either tier, in one pass (fd_rope_store_kv).

    q [T, H, D], k and v [T, KVH, D], one of fp16 / bf16 / fp32; positions
    int64 [A, T] (or [T]): the token's place on each axis; cos_sin fp32
    [max_pos, rot_dim]: cosines of the rot_dim / 2 pairs, then sines; slots
    int64 [T] (-1: not written; the others differ) or None (no KV write).
    sections / turns: which pair takes which axis (rope_axes; default one
    axis).  A pair is dims (i, i + rot_dim / 2), or neighbours (2i, 2i + 1)
    with pairs.  The rotated q goes to q_out (default: q itself), which is
    returned; k_out takes a copy of the rotated k, e.g. for prefill_attn over
    a fresh prompt's own rows."""
    idx, dt = q.get_device(), q.dtype
    if idx < 0:
        raise RuntimeError("q must be a CUDA tensor")
    if q.dim() != 3 or k.dim() != 3:
        raise RuntimeError("q must be [T, H, D], k and v [T, KVH, D]")
    T, H, D = shape = q.shape
    KVH = k.shape[1]
    if k.shape != (T, KVH, D) or v.shape != k.shape:
        raise RuntimeError("q must be [T, H, D], k and v [T, KVH, D]")
    q_out = q if q_out is None else q_out
    if q_out.shape != shape or (k_out is not None and k_out.shape != k.shape):
        raise RuntimeError("q_out / k_out must have q's / k's shape")
    if positions.dim() == 1:
        positions = positions.unsqueeze(0)
    A = 1 if sections is None else len(sections)
    p0, p1 = positions.stride()
    if (positions.dtype is not torch.int64 or positions.get_device() != idx or positions.shape[1] < T
            or (p1 != 1 and T > 1)):
        raise RuntimeError("positions must be int64 [axes, T] on q's device with contiguous rows")
    if positions.shape[0] != A:
        raise RuntimeError("positions must have one row per axis")
    if cos_sin.dtype is not torch.float32 or cos_sin.get_device() != idx or cos_sin.dim() != 2 or not cos_sin.is_contiguous():
        raise RuntimeError("cos_sin must be contiguous fp32 [max_pos, rot_dim] on q's device")
    max_pos, rot = cos_sin.shape
    axes = rope_axes((rot // 2,) if sections is None else tuple(sections), turns)
    if 2 * len(axes) != rot:
        raise RuntimeError("sections must add up to rot_dim / 2 pairs")
    BS, slots_ptr = 0, 0
    f0 = f1 = _NO_TIER
    if slots is not None:
        if slots.dtype is not torch.int64 or slots.get_device() != idx or slots.numel() < T or not slots.is_contiguous():
            raise RuntimeError("slots must be contiguous int64 with T entries on q's device")
        t0, t1 = tiers
        if t0 is None and t1 is None:
            raise RuntimeError("at least one KV tier is required")
        slots_ptr, BS = slots.data_ptr(), (t0 if t0 is not None else t1).k.shape[2]
        f0, f1 = _tier_fields(t0, idx, dt, (KVH, BS, D)), _tier_fields(t1, idx, dt, (KVH, BS, D))
    packed = _ROPE_STRUCT.pack(
        *_rows3(q, idx, dt, "q"), *_rows3(q_out, idx, dt, "q_out"), *_rows3(k, idx, dt, "k"), *_rows3(v, idx, dt, "v"),
        *((0, 0, 0) if k_out is None else _rows3(k_out, idx, dt, "k_out")), positions.data_ptr(), p0, cos_sin.data_ptr(),
        max_pos, slots_ptr, *f0, *f1, tier_split, T, H, KVH, D, rot, BS, dtype_code(dt), A, nat.ROPE_PAIRS if pairs else 0,
        axes, 0, _error_ptr(idx))
    _launch(nat.load().fd_rope_store_kv, packed, idx, "fd_rope_store_kv")
    return q_out


@lru_cache(maxsize=256)
def _attn_workspace_bytes(H: int, KVH: int, D: int, dtype: torch.dtype) -> int:
    a = nat.FdAttnArgs()
    a.num_heads, a.num_kv_heads, a.head_size, a.dtype = H, KVH, D, dtype_code(dtype)
    return nat.load().fd_attn_workspace_size(ctypes.byref(a))


def _attn_fields(q, out, lse, q_start, q_len, k_len, scale, KVH, f0, f1, tier_split, table, W, bt_row, k_start, BS, max_q_len,
                 max_k_len) -> list:
    """The fields of fd_attn_args, its workspace (the third and second last) still 0."""
    idx, dt = q.get_device(), q.dtype
    T, H, D = q.shape
    n = q_len.numel()
    lse_f = (0, 0, 0)
    if lse is not None:
        if lse.dtype is not torch.float32 or lse.get_device() != idx or lse.shape != (H, T):
            raise RuntimeError("lse must be fp32 [H, T] on q's device")
        lse_f = (lse.data_ptr(), *lse.stride())
    return [
        *_rows3(q, idx, dt, "q"), *((0, 0, 0) if out is None else _rows3(out, idx, dt, "out")), *lse_f, *f0, *f1, tier_split,
        *((0, 0) if table is None else (table.data_ptr(), table.stride(0))),
        0 if bt_row is None else _i32(bt_row, idx, n, "bt_row"), 0 if k_start is None else _i32(k_start, idx, n, "k_start"),
        _i32(q_start, idx, n, "q_start"), _i32(q_len, idx, n, "q_len"), _i32(k_len, idx, n, "k_len"), W, T, n, H, KVH, D,
        BS, scale, dtype_code(dt), max_q_len, max_k_len, 0 if table is None else table.shape[0], 0, 0, _error_ptr(idx)]


def _scratch(q: torch.Tensor, workspace_buf: torch.Tensor | None, need: int) -> torch.Tensor:
    if workspace_buf is None:
        return torch.empty(need, dtype=torch.uint8, device=q.device)
    if (workspace_buf.get_device() != q.get_device() or workspace_buf.dtype is not torch.uint8
            or not workspace_buf.is_contiguous() or workspace_buf.numel() < need):
        raise RuntimeError(f"workspace_buf must be contiguous uint8 on q's device with >= {need} bytes")
    return workspace_buf


def _attn(fn, what: str, q, out, lse, q_start, q_len, k_len, scale, KVH, f0, f1, tier_split, table, W, bt_row, k_start, BS,
          max_q_len, max_k_len, workspace_buf) -> None:
    if out.shape != q.shape:
        raise RuntimeError("q and out must be [T, H, D] alike")
    packed = _attn_fields(q, out, lse, q_start, q_len, k_len, scale, KVH, f0, f1, tier_split, table, W, bt_row, k_start, BS,
                          max_q_len, max_k_len)
    if f1[-2]:  # a host tier: its copies count
        need = nat.load().fd_attn_workspace_size(_ATTN_STRUCT.pack(*packed))
    else:
        need = _attn_workspace_bytes(q.shape[1], KVH, q.shape[2], q.dtype)
    buf = _scratch(q, workspace_buf, need)
    packed[-3], packed[-2] = buf.data_ptr(), buf.numel()
    _launch(fn, _ATTN_STRUCT.pack(*packed), q.get_device(), what)


def _paged(q, tiers, block_table, bt_row, n: int) -> tuple:
    """(KVH, BS, C fields of both tiers, W) of a call over the paged cache."""
    t0, t1 = tiers
    if t0 is None and t1 is None:
        raise RuntimeError("at least one KV tier is required")
    idx = q.get_device()
    if idx < 0:
        raise RuntimeError("q must be a CUDA tensor")
    _, KVH, BS, D = (t0 if t0 is not None else t1).k.shape
    if q.dim() != 3 or q.shape[2] != D:
        raise RuntimeError("q must be [T, H, D] with the cache's head size")
    if block_table.dtype is not torch.int32 or block_table.get_device() != idx or block_table.dim() != 2:
        raise RuntimeError("block_table must be int32 [R, W] on q's device")
    R, W = block_table.shape
    if W > 1 and block_table.stride(1) != 1:
        raise RuntimeError("block_table rows must be contiguous")
    if bt_row is None and R < n:
        raise RuntimeError("block_table must have a row per request")
    return KVH, BS, _tier_fields(t0, idx, q.dtype, (KVH, BS, D)), _tier_fields(t1, idx, q.dtype, (KVH, BS, D)), W


def chunk_attn(q: torch.Tensor, tiers: tuple[KVTier | None, KVTier | None], tier_split: int, block_table: torch.Tensor,
               q_start: torch.Tensor, q_len: torch.Tensor, k_len: torch.Tensor, scale: float, out: torch.Tensor,
               lse: torch.Tensor | None = None, *, bt_row: torch.Tensor | None = None, max_q_len: int = 0,
               max_k_len: int = 0, workspace_buf: torch.Tensor | None = None) -> None:
    """Attention of each request's new tokens over its paged cache in both
    tiers (fd_chunk_attn): chunks of prompts, draft tokens to verify, single
    tokens.  Unlike prefill_attn it reads the host tier too, takes head sizes
    up to 256 (of whole 16 bytes) and any block size and dtype, splits long contexts over the GPU when there
    are few queries, and returns the log-sum-exp.

    q, out [T, H, D]; per request (int32 [n] on the device) q_start, q_len,
    k_len: its queries are rows q_start .. of q and its K/V, the new tokens'
    included, k_len tokens in the blocks of row bt_row[r] (default r; a row
    outside the table: the request writes nothing and raises the error word) of
    block_table [R, W] int32; query i sees keys 0 .. k_len - q_len + i.  lse
    fp32 [H, T] or None.  Rows of no request stay as they were; a query that
    sees nothing gets 0 and -inf.  max_q_len / max_k_len: the lengths' bounds,
    if the host knows them.  workspace_buf (uint8) replaces the call's own
    scratch memory."""
    KVH, BS, f0, f1, W = _paged(q, tiers, block_table, bt_row, q_len.numel())
    _attn(nat.load().fd_chunk_attn, "fd_chunk_attn", q, out, lse, q_start, q_len, k_len, scale, KVH, f0, f1, tier_split,
          block_table, W, bt_row, None, BS, max_q_len, max_k_len, workspace_buf)


def cross_attn(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_start: torch.Tensor, q_len: torch.Tensor,
               k_start: torch.Tensor, k_len: torch.Tensor, scale: float, out: torch.Tensor,
               lse: torch.Tensor | None = None, *, max_q_len: int = 0, max_k_len: int = 0,
               workspace_buf: torch.Tensor | None = None) -> None:
    """Cross attention to an encoder's states (fd_cross_attn): request r's
    queries (rows q_start .. q_start + q_len - 1 of q [T, H, D]) each see all
    of rows k_start .. k_start + k_len - 1 of k and v [S, KVH, D]; requests may
    share states.  q_len = 1 is a decode step.  The other arguments are
    chunk_attn's."""
    idx, dt = q.get_device(), q.dtype
    if idx < 0:
        raise RuntimeError("q must be a CUDA tensor")
    if q.dim() != 3 or k.dim() != 3 or k.shape != v.shape or k.stride() != v.stride() or k.shape[2] != q.shape[2]:
        raise RuntimeError("k and v must be [S, KVH, D] alike with q's head size")
    S, KVH, _ = k.shape
    k_ptr, k_st, k_sh = _rows3(k, idx, dt, "k")
    _attn(nat.load().fd_cross_attn, "fd_cross_attn", q, out, lse, q_start, q_len, k_len, scale, KVH,
          (k_ptr, _rows3(v, idx, dt, "v")[0], 0, k_sh, k_st, S, 0, 0), _NO_TIER, 0, None, 0, None, k_start, 0, max_q_len,
          max_k_len, workspace_buf)


# ------------------------------------------------------------- after the attention


@dataclass(frozen=True)
class KeyStats:
    """What each cached key of one layer has received: weights fp32 and
    positions int32, both contiguous [blocks, KVH, block_size] on the device and
    indexed by block id, host-tier blocks included."""

    weights: torch.Tensor
    positions: torch.Tensor

    def __post_init__(self) -> None:
        w, p = self.weights, self.positions
        _check(w.dim() == 3 and w.shape == p.shape, "weights and positions must be [blocks, KVH, block_size] alike")
        _check(w.dtype == torch.float32 and p.dtype == torch.int32, "weights must be float32, positions int32")
        _check(w.is_contiguous() and p.is_contiguous() and w.is_cuda and p.device == w.device,
               "weights and positions must be contiguous on one CUDA device")

    @classmethod
    def zeros(cls, num_blocks: int, num_kv_heads: int, block_size: int, device) -> "KeyStats":
        shape = (num_blocks, num_kv_heads, block_size)
        return cls(torch.zeros(shape, dtype=torch.float32, device=device), torch.zeros(shape, dtype=torch.int32, device=device))

    def _fields(self, idx: int, KVH: int, BS: int) -> tuple:
        w = self.weights
        B, h, b = w.shape
        if w.get_device() != idx or h != KVH or b != BS:
            raise RuntimeError("stats must be [blocks, KVH, block_size] of the cache on the call's device")
        return w.data_ptr(), self.positions.data_ptr(), B


class KeyMoves(_Buffers):
    """Device buffers that select_keys fills and move_keys reads, for R requests
    of KVH kv heads and up to `room` moves each: src and dst int32 [R, KVH,
    room], counts int32 [R, KVH].  A request cut from n keys to b needs room for
    min(b, n - b)."""

    def __init__(self, R: int, KVH: int, room: int, device, src: torch.Tensor | None = None,
                 dst: torch.Tensor | None = None, counts: torch.Tensor | None = None):
        lists = (R, KVH, room)
        super().__init__(device, src=(lists if src is None else src, R * KVH * room),
                         dst=(lists if dst is None else dst, R * KVH * room),
                         counts=((R, KVH) if counts is None else counts, R * KVH))
        self.__dict__.update(R=int(R), KVH=int(KVH), room=int(room))

    def _fields(self, idx: int, R: int, KVH: int) -> tuple:
        if self.KVH != KVH or self.R < R or self.idx != idx:
            raise RuntimeError("moves must be of at least R requests and of KVH kv heads, on the call's device")
        return self.src.data_ptr(), self.dst.data_ptr(), self.counts.data_ptr()


def key_weights(q: torch.Tensor, tiers: tuple[KVTier | None, KVTier | None], tier_split: int, block_table: torch.Tensor,
                q_start: torch.Tensor, q_len: torch.Tensor, k_len: torch.Tensor, scale: float, lse: torch.Tensor,
                stats: KeyStats, *, evicted: torch.Tensor | None = None, bt_row: torch.Tensor | None = None,
                max_q_len: int = 0, max_k_len: int = 0, workspace_buf: torch.Tensor | None = None) -> None:
    """Add up the attention weight that each cached key receives in a step
    (fd_key_weights): over the queries that see it and the heads of its kv head,
    exp(scale q.k - lse), with lse [H, T] as chunk_attn (or the decode) wrote
    it.  The other arguments are chunk_attn's.

    The q_len newest keys of a request are new: their weight in `stats` is set,
    whatever it was, and their position becomes their index plus evicted[r]
    (int32 [n], see trim_tables).  Older keys' weights are added to.  So a key
    needs no reset when its block is handed to another request, and a step whose
    drafts were rejected can count the accepted ones alone (q_len and k_len
    without the others).  A key that no call had among the newest keeps the weight
    and the position that its place held before, so a prompt's tokens count
    whole."""
    KVH, BS, f0, f1, W = _paged(q, tiers, block_table, bt_row, q_len.numel())
    idx = q.get_device()
    lib = nat.load()
    fields = _attn_fields(q, None, lse, q_start, q_len, k_len, scale, KVH, f0, f1, tier_split, block_table, W, bt_row, None, BS,
                          max_q_len, max_k_len)
    more = (*stats._fields(idx, KVH, BS), 0 if evicted is None else _i32(evicted, idx, q_len.numel(), "evicted"))
    packed = _KEY_WEIGHTS_STRUCT.pack(*fields, *more)
    need = lib.fd_key_weights_workspace_size(packed)
    if need > 0 or workspace_buf is not None:
        buf = _scratch(q, workspace_buf, need)
        fields[-3], fields[-2] = buf.data_ptr(), buf.numel()
        packed = _KEY_WEIGHTS_STRUCT.pack(*fields, *more)
    _launch(lib.fd_key_weights, packed, idx, "fd_key_weights")


def select_keys(stats: KeyStats, block_table: torch.Tensor, seq_lens: torch.Tensor, keep_lens: torch.Tensor,
                moves: KeyMoves | None = None, *, sinks: int = 0, recent: int = 0, evicted: torch.Tensor | None = None,
                max_k_len: int = 0) -> KeyMoves:
    """Choose the keys that stay when caches are cut to a budget
    (fd_select_keys), per request and kv head: those whose position is below
    `sinks` or among the newest `recent`, then those with the most weight, the
    lowest index first where weights are equal (a NaN is the least).

    seq_lens int32 [R]: the tokens in the cache; keep_lens int32 [R]: those to
    keep (below 0, or not below seq_lens: the request is left as it is);
    evicted int32 [R]: tokens cut earlier.  Writes to `moves` (default: a new
    one, with room for max_k_len / 2 moves) which keys move where, all from
    behind the budget to before it; nothing else changes.  A request that could
    need more moves than there is room for has none, and sets the error word.
    max_k_len: the host's bound on seq_lens, if it knows one (0: what the table's
    rows hold).  With `moves` given it only chooses the launch, and a wrong one
    costs time, not the result; without, it also sizes the new one, and has to
    hold."""
    idx, R, W = _block_table(block_table)
    _, KVH, BS = stats.weights.shape
    if moves is None:
        moves = KeyMoves(R, KVH, (max_k_len if max_k_len > 0 else W * BS) // 2, block_table.device)
    packed = _SELECT_STRUCT.pack(
        *stats._fields(idx, KVH, BS), block_table.data_ptr(), block_table.stride(0), _i32(seq_lens, idx, R, "seq_lens"),
        _i32(keep_lens, idx, R, "keep_lens"), 0 if evicted is None else _i32(evicted, idx, R, "evicted"),
        *moves._fields(idx, R, KVH), W, R, KVH, BS, moves.room, sinks, recent, max_k_len, _error_ptr(idx))
    _launch(nat.load().fd_select_keys, packed, idx, "fd_select_keys")
    return moves


def move_keys(moves: KeyMoves, tiers: tuple[KVTier | None, KVTier | None], tier_split: int, block_table: torch.Tensor,
              stats: KeyStats | None = None) -> None:
    """Move the K and V rows that `moves` lists within each request's blocks, in
    either tier, and their weights and positions in `stats` (fd_move_keys).  Then
    the first keep_lens tokens of each request are its cache (trim_tables, once
    all layers have moved theirs).  K rows carry their rotary positions with
    them, so their order within the cache does not matter to the queries that
    come after."""
    t0, t1 = tiers
    if t0 is None and t1 is None:
        raise RuntimeError("at least one KV tier is required")
    idx, R, W = _block_table(block_table)
    k = (t0 if t0 is not None else t1).k
    _, KVH, BS, D = k.shape
    shape = (KVH, BS, D)
    packed = _MOVE_STRUCT.pack(
        *moves._fields(idx, R, KVH), *_tier_fields(t0, idx, k.dtype, shape), *_tier_fields(t1, idx, k.dtype, shape), tier_split,
        block_table.data_ptr(), block_table.stride(0), *((0, 0, 0) if stats is None else stats._fields(idx, KVH, BS)), W, R,
        KVH, D, BS, moves.room, dtype_code(k.dtype), 0, _error_ptr(idx))
    _launch(nat.load().fd_move_keys, packed, idx, "fd_move_keys")


class DraftVerdict(_Buffers):
    """Device buffers that verify_drafts fills for R requests of up to K drafted
    tokens: tokens int64 [R, K + 1] (the accepted drafts, the token that
    follows, then -1), accepted int32 [R], keep_lens int32 [R] (-1, which
    trim_tables leaves alone, until a call that is given seq_lens)."""

    def __init__(self, R: int, K: int, device):
        super().__init__(device, accepted=(R, R), keep_lens=(torch.full((R,), -1, dtype=torch.int32, device=device), R))
        self.__dict__.update(R=int(R), K=int(K), tokens=torch.full((R, K + 1), -1, dtype=torch.int64, device=device))


def verify_drafts(target_probs: torch.Tensor, draft_tokens: torch.Tensor, draft_probs: torch.Tensor | None,
                  q_start: torch.Tensor, q_len: torch.Tensor, accept_u: torch.Tensor, sample_u: torch.Tensor, *,
                  seq_lens: torch.Tensor | None = None, out: DraftVerdict | None = None) -> DraftVerdict:
    """Verify drafted tokens against the target's probabilities and draw the
    token that follows the accepted ones (fd_verify_drafts); q_len = 1 is
    ordinary sampling.

    target_probs [T, V]: a row per query of the step; q_start, q_len int32 [R]
    as extend_tables gives them (q_len = 1 + drafts; 0: no part in the step), or,
    where a request's new tokens are a prompt's, its last row and 1;
    draft_tokens int64 [R, K]; draft_probs [R, K, V] of target_probs' dtype
    (fp32, fp16 or bf16), or None where the draft is no distribution;
    accept_u fp32 [R, K] and sample_u fp32 [R]: uniform numbers in [0, 1).
    Draft d is accepted while accept_u q < p; the token after the accepted ones
    comes from max(p - q, 0) of the rejected draft, or from the last row, by
    sample_u's place in the running sum.  A one-hot row is greedy decoding.
    Fills and returns `out`; keep_lens, with seq_lens int32 [R] (the drafts
    included), is the cache that stays: trim_tables' keep_lens.  Without
    seq_lens, keep_lens is left as it was."""
    idx, dt = target_probs.get_device(), target_probs.dtype
    if idx < 0:
        raise RuntimeError("target_probs must be a CUDA tensor")
    if target_probs.dim() != 2 or (target_probs.stride(1) != 1 and target_probs.shape[1] != 1):
        raise RuntimeError("target_probs must be [T, V] with contiguous rows")
    T, V = target_probs.shape
    if draft_tokens.dim() != 2 or draft_tokens.dtype is not torch.int64 or draft_tokens.get_device() != idx or (
            draft_tokens.stride(1) != 1 and draft_tokens.shape[1] > 1):
        raise RuntimeError("draft_tokens must be int64 [R, K] with contiguous rows on target_probs' device")
    R, K = draft_tokens.shape
    if accept_u.shape != (R, K) or accept_u.dtype is not torch.float32 or accept_u.get_device() != idx or (
            accept_u.stride(1) != 1 and K > 1):
        raise RuntimeError("accept_u must be fp32 [R, K] with contiguous rows on target_probs' device")
    if sample_u.dtype is not torch.float32 or sample_u.get_device() != idx or sample_u.numel() < R or not sample_u.is_contiguous():
        raise RuntimeError("sample_u must be contiguous fp32 [R] on target_probs' device")
    probs = (0, 0, 0)
    if draft_probs is not None:
        if draft_probs.shape != (R, K, V) or draft_probs.dtype is not dt or draft_probs.get_device() != idx or (
                draft_probs.stride(2) != 1 and V > 1):
            raise RuntimeError("draft_probs must be [R, K, V] with contiguous rows and target_probs' dtype and device")
        probs = (draft_probs.data_ptr(), draft_probs.stride(0), draft_probs.stride(1))
    if out is None:
        out = DraftVerdict(R, K, target_probs.device)
    if out.R < R or out.K != K or out.idx != idx:
        raise RuntimeError("out must be a DraftVerdict of at least R requests and of K drafts on target_probs' device")
    packed = _VERIFY_STRUCT.pack(
        target_probs.data_ptr(), target_probs.stride(0), *probs, draft_tokens.data_ptr(), draft_tokens.stride(0),
        _i32(q_start, idx, R, "q_start"), _i32(q_len, idx, R, "q_len"), accept_u.data_ptr(), accept_u.stride(0),
        sample_u.data_ptr(), 0 if seq_lens is None else _i32(seq_lens, idx, R, "seq_lens"), out.tokens.data_ptr(),
        out.accepted.data_ptr(), out.keep_lens.data_ptr(), R, K, V, T, dtype_code(dt), 0, _error_ptr(idx))
    _launch(nat.load().fd_verify_drafts, packed, idx, "fd_verify_drafts")
    return out


# ------------------------------------------------------------- merge


def merge_attn_states(out: torch.Tensor, o_a: torch.Tensor, lse_a: torch.Tensor, o_b: torch.Tensor,
                      lse_b: torch.Tensor, out_lse: torch.Tensor | None = None,
                      out_rows: torch.Tensor | None = None) -> None:
    """vLLM merge_attn_states(output, prefix_output, prefix_lse, suffix_output,
    suffix_lse) with the reference's rule (fastdecode/cpu_ops.py:93-113).
    o_a/o_b [n,H,D] contiguous, lse [H,n] fp32; out rows out_rows[i] or i."""
    _check(o_a.shape == o_b.shape and o_a.dtype == o_b.dtype, "o_a and o_b must match")
    _check(o_a.is_contiguous() and o_b.is_contiguous(), "partials must be contiguous")
    n, H, D = o_a.shape
    _check(lse_a.shape == (H, n) and lse_b.shape == (H, n), "lse must be [H, n]")
    _check(lse_a.dtype == torch.float32 and lse_b.dtype == torch.float32, "lse must be float32")
    _check(lse_a.is_contiguous() and lse_b.is_contiguous(), "lse must be contiguous")
    _check(out.stride(-1) == 1 and out.stride(1) == D, "out rows must be [H, D] contiguous")
    dev = o_a.device
    if out_rows is not None:  # read as int64 by the kernel
        _check(out_rows.dtype == torch.int64 and out_rows.device == dev and out_rows.is_contiguous()
               and out_rows.numel() >= n, "out_rows must be a contiguous int64 tensor on the device with n entries")
    nat.check(nat.load().fd_merge_attn_states(
        out.data_ptr(), dtype_code(out.dtype), out.stride(0), _ptr(out_rows), _ptr(out_lse),
        o_a.data_ptr(), lse_a.data_ptr(), o_b.data_ptr(), lse_b.data_ptr(), dtype_code(o_a.dtype),
        n, H, D, _stream(dev)), "fd_merge_attn_states")


def merge_partials(parts: torch.Tensor, num_parts: int, n: int, H: int, D: int, out: torch.Tensor,
                   out_lse: torch.Tensor | None = None) -> None:
    """P-way merge of packed fp32 partials: part p occupies parts[p] =
    [o (n*H*D) | lse (H*n)]."""
    _check(parts.dtype == torch.float32 and parts.is_contiguous(), "parts must be contiguous fp32")
    stride = n * H * D + H * n
    _check(parts.numel() >= num_parts * stride, "parts buffer too small")
    _check(out.is_contiguous() and out.shape == (n, H, D), "out must be [n, H, D] contiguous")
    base = parts.data_ptr()
    nat.check(nat.load().fd_merge_partials(
        base, base + 4 * n * H * D, stride, num_parts, n, H, D, out.data_ptr(), dtype_code(out.dtype),
        _ptr(out_lse), _stream(parts.device)), "fd_merge_partials")


# ------------------------------------------------------------- load_ext shim


class _Ext:
    """Object returned by load_ext(), shaped like the reference's pybind
    module (fastdecode/csrc/cpu_attn.cpp:531-537)."""

    decode_attn = staticmethod(decode_attn)
    store_kv = staticmethod(store_kv)
    merge_attn_states = staticmethod(merge_attn_states)

    @staticmethod
    def set_num_threads(n: int) -> None:  # the GPU path has no host thread pool
        del n

    @staticmethod
    def get_num_threads() -> int:
        return 1

    @staticmethod
    def has_avx2() -> bool:  # no host SIMD kernel exists in this engine
        return False


def load_ext(verbose: bool = False) -> _Ext:
    """Load the native library; raises if it is missing (no fallback)."""
    del verbose
    nat.load()
    return _Ext()
