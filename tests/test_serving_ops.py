"""Refusals and host-side arithmetic of the operators behind a step's attention
(key_weights, select_keys, move_keys, trim_tables, verify_drafts): every bad
argument is reported before anything is launched, so no GPU is needed here."""

from __future__ import annotations

import ctypes

import pytest
import torch

from vllm_fastdecoder_b200 import _native as nat
from vllm_fastdecoder_b200 import gpu_ops

PAIRS = [(nat.FdTrimArgs, "_TRIM_STRUCT", "fd_trim_args_bytes"), (nat.FdVerifyArgs, "_VERIFY_STRUCT", "fd_verify_args_bytes"),
         (nat.FdKeyWeightsArgs, "_KEY_WEIGHTS_STRUCT", "fd_key_weights_args_bytes"),
         (nat.FdSelectArgs, "_SELECT_STRUCT", "fd_select_args_bytes"), (nat.FdMoveArgs, "_MOVE_STRUCT", "fd_move_args_bytes")]


def _number(a, start, want):
    """A different number in every scalar of struct `a`, and those numbers in order."""
    for name, typ in a._fields_:
        if isinstance(typ, type) and issubclass(typ, ctypes.Structure):
            start = _number(getattr(a, name), start, want)
        elif hasattr(typ, "_length_"):
            arr = getattr(a, name)
            for k in range(typ._length_):
                if issubclass(typ._type_, ctypes.Structure):
                    start = _number(arr[k], start, want)
                else:
                    start += 1
                    arr[k] = start
                    want.append(start)
        else:
            start += 1
            setattr(a, name, start)
            want.append(start)
    return start


@pytest.mark.parametrize("mirror,packer,size", PAIRS)
def test_struct_mirrors_and_packers_match_the_library(mirror, packer, size):
    s = getattr(gpu_ops, packer)
    assert getattr(nat.load(), size)() == ctypes.sizeof(mirror) == s.size
    a, want = mirror(), []
    _number(a, 0, want)
    assert bytes(a) == s.pack(*want)


def test_version_and_new_device_errors():
    lib = nat.load()
    assert lib.fd_version() >= 104
    assert b"vocabulary" in lib.fd_device_error_string(9) and b"probability" in lib.fd_device_error_string(10)


def _trim():
    a = nat.FdTrimArgs()
    for f in ("keep_lens", "lens_in", "lens_out", "block_table", "counts_in", "counts_out", "header"):
        setattr(a, f, 4096)
    a.free_ids[0], a.free_ids[1] = 4096, 4096
    a.free_cap[0] = a.free_cap[1] = 10
    a.bt_stride = a.bt_width = 4
    a.num_reqs, a.num_gpu_blocks, a.num_cpu_blocks, a.block_size = 3, 8, 8, 16
    return a


@pytest.mark.parametrize("field,value,code,msg", [
    ("num_reqs", -1, 1, b"num_reqs"), ("block_size", 0, 1, b"block_size"), ("num_gpu_blocks", -1, 1, b"block counts"),
    ("num_cpu_blocks", -1, 1, b"block counts"), ("num_reqs", 8193, 2, b"at most 8192"), ("num_gpu_blocks", 1 << 31, 2, b"int32"),
    ("bt_width", 0, 1, b"bt_width"), ("bt_stride", -1, 1, b"bt_stride"), ("bt_width", 1 << 28, 2, b"int32"),
    ("keep_lens", None, 1, b"null"), ("lens_in", None, 1, b"null"), ("lens_out", None, 1, b"null"), ("block_table", None, 1, b"null"),
    ("counts_in", None, 1, b"null"), ("counts_out", None, 1, b"null"), ("header", None, 1, b"null"),
])
def test_trim_rejects_bad_arguments(field, value, code, msg):
    a = _trim()
    setattr(a, field, value)
    assert nat.load().fd_trim_tables(ctypes.byref(a), None) == code
    assert msg in nat.load().fd_last_error_message()


def test_trim_rejects_stacks_without_memory():
    for t, cap, ptr in ((0, -1, 4096), (1, 5, None)):
        a = _trim()
        a.free_cap[t], a.free_ids[t] = cap, ptr
        assert nat.load().fd_trim_tables(ctypes.byref(a), None) == 1
        assert b"no memory" in nat.load().fd_last_error_message()


def _verify():
    a = nat.FdVerifyArgs()
    for f in ("target", "draft_probs", "draft_tokens", "q_start", "q_len", "accept_u", "sample_u", "lens", "tokens", "accepted",
              "keep_lens"):
        setattr(a, f, 4096)
    a.target_stride = a.draft_stride_k = 100
    a.num_reqs, a.num_drafts, a.vocab, a.num_rows, a.dtype = 2, 3, 100, 8, 2
    return a


@pytest.mark.parametrize("field,value,code,msg", [
    ("dtype", 5, 2, b"dtype"), ("num_reqs", -1, 1, b"num_reqs"), ("num_drafts", -1, 1, b"num_drafts"), ("vocab", 0, 1, b"vocab"),
    ("num_rows", -1, 1, b"num_rows"), ("num_drafts", 1025, 2, b"at most 1024"), ("num_reqs", (1 << 24) + 1, 2, b"requests"),
    ("target", None, 1, b"null"), ("q_start", None, 1, b"null"), ("q_len", None, 1, b"null"), ("sample_u", None, 1, b"null"),
    ("accept_u", None, 1, b"null"), ("draft_tokens", None, 1, b"null"), ("tokens", None, 1, b"null"), ("accepted", None, 1, b"null"),
    ("keep_lens", None, 1, b"null"), ("target_stride", 99, 1, b"overlap"),
])
def test_verify_rejects_bad_arguments(field, value, code, msg):
    a = _verify()
    setattr(a, field, value)
    assert nat.load().fd_verify_drafts(ctypes.byref(a), None) == code
    assert msg in nat.load().fd_last_error_message()


def test_verify_of_no_requests_is_nothing():
    a = _verify()
    a.num_reqs = 0
    assert nat.load().fd_verify_drafts(ctypes.byref(a), None) == 0


def _weights():
    a = nat.FdKeyWeightsArgs()
    t = a.attn
    t.q = t.lse = t.block_table = t.q_start = t.q_len = t.k_len = 4096
    t.q_stride_t, t.q_stride_h = 256, 64
    t.tier[0].k = t.tier[0].v = 4096
    t.tier[0].blk_stride, t.tier[0].head_stride, t.tier[0].tok_stride, t.tier[0].num_blocks = 2048, 1024, 64, 8
    t.tier_split, t.bt_stride, t.bt_width, t.bt_rows = 8, 4, 4, 2
    t.num_tokens, t.n, t.num_heads, t.num_kv_heads, t.head_size, t.block_size = 2, 2, 4, 2, 64, 16
    t.scale, t.dtype = 0.125, 1
    a.stats.weights = a.stats.positions = 4096
    a.stats.num_blocks = 8
    return a


@pytest.mark.parametrize("field,value,code,msg", [
    ("dtype", 7, 2, b"dtype"), ("n", -1, 1, b"negative"), ("num_tokens", -1, 1, b"negative"), ("n", 65536, 2, b"65535"),
    ("num_kv_heads", 0, 1, b"multiple"), ("num_heads", 5, 1, b"multiple"), ("num_heads", 130, 2, b"group"), ("head_size", 0, 2, b"256"),
    ("head_size", 264, 2, b"256"), ("head_size", 68, 3, b"16"), ("scale", 0.0, 1, b"scale"), ("lse", None, 1, b"lse"),
    ("q", None, 1, b"required"), ("k_len", None, 1, b"required"), ("block_table", None, 1, b"block_table"),
    ("block_size", 0, 1, b"block_size"), ("bt_rows", -1, 1, b"bt_rows"), ("q", 4100, 3, b"aligned"), ("q_stride_h", 60, 3, b"aligned"),
])
def test_key_weights_rejects_bad_arguments(field, value, code, msg):
    a = _weights()
    setattr(a.attn, field, value)
    assert nat.load().fd_key_weights(ctypes.byref(a), None) == code
    assert msg in nat.load().fd_last_error_message()


def test_key_weights_rejects_bad_stats_and_workspace():
    lib = nat.load()
    for field, value in (("weights", None), ("positions", None), ("num_blocks", -1)):
        a = _weights()
        setattr(a.stats, field, value)
        assert lib.fd_key_weights(ctypes.byref(a), None) == 1
        assert b"stats" in lib.fd_last_error_message()
    a = _weights()  # many rows over unknown lengths: items are cut, and that needs memory
    a.attn.num_tokens, a.attn.dtype = 5000, 1
    assert lib.fd_key_weights_workspace_size(ctypes.byref(a)) > 0
    assert lib.fd_key_weights(ctypes.byref(a), None) == 4
    assert b"workspace" in lib.fd_last_error_message()


def test_key_weights_workspace_is_for_cut_items_and_host_copies():
    lib = nat.load()
    a = _weights()
    assert lib.fd_key_weights_workspace_size(ctypes.byref(a)) == 0  # single tokens: items stay whole
    a.attn.tier[1].host_mapped, a.attn.tier[1].num_blocks = 1, 4
    assert lib.fd_key_weights_workspace_size(ctypes.byref(a)) > 0
    a.attn.num_kv_heads = 0
    assert lib.fd_key_weights_workspace_size(ctypes.byref(a)) == 0


@pytest.mark.parametrize("heads,kv_heads", [(4, 2), (32, 1), (64, 1)])
@pytest.mark.parametrize("tokens,n", [(0, 2), (2, 0), (0, 0), (-1, 2), (2, -1)])
@pytest.mark.parametrize("dtype,D", [(1, 64), (0, 128), (2, 64)])
def test_key_weights_of_an_empty_step_needs_nothing(dtype, D, tokens, n, heads, kv_heads):
    """No scratch memory, and no arithmetic on chunks of no rows (more heads per kv head than the fewest columns)."""
    lib = nat.load()
    a = _weights()
    t = a.attn
    t.num_tokens, t.n, t.num_heads, t.num_kv_heads, t.head_size, t.dtype = tokens, n, heads, kv_heads, D, dtype
    t.q_stride_h, t.q_stride_t = D, heads * D
    t.tier[1].host_mapped, t.tier[1].num_blocks = 1, 4
    assert lib.fd_key_weights_workspace_size(ctypes.byref(a)) == 0
    assert lib.fd_key_weights(ctypes.byref(a), None) == (0 if tokens >= 0 and n >= 0 else 1)


def _select():
    a = nat.FdSelectArgs()
    a.stats.weights = a.stats.positions = 4096
    a.stats.num_blocks = 8
    for f in ("block_table", "lens", "keep_lens", "src", "dst", "counts"):
        setattr(a, f, 4096)
    a.bt_stride = a.bt_width = 4
    a.num_reqs, a.num_kv_heads, a.block_size, a.room = 2, 2, 16, 8
    return a


@pytest.mark.parametrize("field,value,code,msg", [
    ("num_reqs", -1, 1, b"num_reqs"), ("num_kv_heads", 0, 1, b"num_kv_heads"), ("block_size", 0, 1, b"block_size"),
    ("room", -1, 1, b"room"), ("sinks", -1, 1, b"sinks"), ("recent", -1, 1, b"recent"), ("num_reqs", 65536, 2, b"65535"),
    ("num_kv_heads", 5000, 2, b"4096"), ("bt_width", 0, 1, b"bt_width"), ("bt_stride", -1, 1, b"bt_stride"),
    ("bt_width", 1 << 27, 2, b"int32"), ("block_table", None, 1, b"null"), ("lens", None, 1, b"null"), ("keep_lens", None, 1, b"null"),
    ("counts", None, 1, b"null"), ("src", None, 1, b"null"), ("dst", None, 1, b"null"),
])
def test_select_rejects_bad_arguments(field, value, code, msg):
    a = _select()
    setattr(a, field, value)
    assert nat.load().fd_select_keys(ctypes.byref(a), None) == code
    assert msg in nat.load().fd_last_error_message()


def _move():
    a = nat.FdMoveArgs()
    for f in ("src", "dst", "counts", "block_table"):
        setattr(a, f, 4096)
    a.tier[0].k = a.tier[0].v = 4096
    a.tier[0].blk_stride, a.tier[0].head_stride, a.tier[0].tok_stride, a.tier[0].num_blocks = 2048, 1024, 64, 8
    a.stats.weights = a.stats.positions = 4096
    a.stats.num_blocks = 8
    a.bt_stride = a.bt_width = 4
    a.num_reqs, a.num_kv_heads, a.head_size, a.block_size, a.room, a.dtype = 2, 2, 64, 16, 8, 1
    return a


@pytest.mark.parametrize("field,value,code,msg", [
    ("dtype", 3, 2, b"dtype"), ("num_reqs", -1, 1, b"num_reqs"), ("num_kv_heads", 0, 1, b"num_kv_heads"), ("head_size", 0, 1, b"head_size"),
    ("block_size", 0, 1, b"block_size"), ("room", -1, 1, b"room"), ("num_reqs", 65536, 2, b"65535"), ("head_size", 68, 3, b"16"),
    ("head_size", 65544, 2, b"65536"), ("bt_width", 0, 1, b"bt_width"), ("src", None, 1, b"null"), ("dst", None, 1, b"null"),
    ("counts", None, 1, b"null"), ("block_table", None, 1, b"null"),
])
def test_move_rejects_bad_arguments(field, value, code, msg):
    a = _move()
    setattr(a, field, value)
    assert nat.load().fd_move_keys(ctypes.byref(a), None) == code
    assert msg in nat.load().fd_last_error_message()


def test_move_rejects_bad_tiers_and_stats():
    lib = nat.load()
    for change, code, msg in ((lambda a: setattr(a.tier[0], "k", None), 1, b"no K/V"), (lambda a: setattr(a.tier[0], "v", 4104), 3, b"aligned"),
                              (lambda a: setattr(a.tier[0], "tok_stride", 60), 3, b"aligned"),
                              (lambda a: setattr(a.stats, "positions", None), 1, b"null")):
        a = _move()
        change(a)
        assert lib.fd_move_keys(ctypes.byref(a), None) == code
        assert msg in lib.fd_last_error_message()


def test_buffers_are_checked_when_made_and_stay():
    i32 = lambda *n: torch.zeros(n, dtype=torch.int32)  # noqa: E731
    for bad in (dict(src=i32(2, 3, 3)), dict(dst=torch.zeros(2, 3, 4)), dict(counts=i32(6, 2)[:, 0])):
        with pytest.raises(RuntimeError, match=next(iter(bad))):
            gpu_ops.KeyMoves(2, 3, 4, "cpu", **bad)
    with pytest.raises(RuntimeError, match="seq_lens"):
        gpu_ops.TrimTables(5, "cpu", seq_lens=i32(4))
    for made, name in ((gpu_ops.KeyMoves(2, 3, 4, "cpu"), "src"), (gpu_ops.TrimTables(2, "cpu"), "seq_lens"),
                       (gpu_ops.DraftVerdict(2, 3, "cpu"), "tokens")):
        with pytest.raises(AttributeError, match="bound again"):
            setattr(made, name, i32(99))
    with pytest.raises(RuntimeError, match="CUDA device"):
        gpu_ops.KeyStats(torch.zeros(2, 3, 4), i32(2, 3, 4))


def test_a_verdict_s_lengths_leave_requests_alone_until_they_are_filled():
    """verify_drafts writes keep_lens where it is given the lengths; trim_tables leaves a request below 0 as it is."""
    v = gpu_ops.DraftVerdict(3, 2, "cpu")
    assert v.keep_lens.tolist() == [-1] * 3 and v.keep_lens.dtype is torch.int32
    assert v.accepted.tolist() == [0] * 3 and v.tokens.tolist() == [[-1] * 3] * 3
    assert gpu_ops.DraftVerdict(0, 2, "cpu").keep_lens.numel() == 0


def test_calls_refuse_host_tensors():
    i32 = lambda *n: torch.zeros(n, dtype=torch.int32)  # noqa: E731
    free = gpu_ops.FreeBlocks(i32(4), None, i32(2))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        gpu_ops.trim_tables(i32(2), i32(2), i32(2, 4), free, 8, 0, 16)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        gpu_ops.verify_drafts(torch.zeros(4, 10), torch.zeros(2, 1, dtype=torch.int64), None, i32(2), i32(2), torch.zeros(2, 1),
                              torch.zeros(2))
    tier = gpu_ops.KVTier(torch.zeros(4, 2, 16, 64), torch.zeros(4, 2, 16, 64))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        gpu_ops.move_keys(gpu_ops.KeyMoves(2, 2, 4, "cpu"), (tier, None), 4, i32(2, 4))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        gpu_ops.key_weights(torch.zeros(2, 4, 64), (tier, None), 4, i32(2, 4), i32(2), i32(2), i32(2), 0.125, torch.zeros(4, 2), None)
