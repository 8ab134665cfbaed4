"""Refusals and host-side arithmetic of the multi-token step's operators
(extend_tables, rope_store_kv, chunk_attn, cross_attn): every bad argument is
reported before anything is launched, so no GPU is needed here."""

from __future__ import annotations

import ctypes

import pytest
import torch

from vllm_fastdecoder_b200 import _native as nat
from vllm_fastdecoder_b200 import gpu_ops, kernel_bench


def test_struct_mirrors_and_packers_match_the_library():
    lib = nat.load()
    for size, mirror, packer in ((lib.fd_tables_args_bytes(), nat.FdTablesArgs, gpu_ops._TABLES_STRUCT),
                                 (lib.fd_rope_args_bytes(), nat.FdRopeArgs, gpu_ops._ROPE_STRUCT),
                                 (lib.fd_attn_args_bytes(), nat.FdAttnArgs, gpu_ops._ATTN_STRUCT)):
        assert size == ctypes.sizeof(mirror) == packer.size


def _numbered(mirror):
    """The mirror with a different number in every scalar, and those numbers in order."""
    a, want, i = mirror(), [], 0
    for name, typ in mirror._fields_:
        if typ in (nat.FdKvTier * 2,):
            for t in getattr(a, name):
                for f, _ in t._fields_:
                    i += 1
                    setattr(t, f, i)
                    want.append(i)
        elif hasattr(typ, "_length_"):
            if typ is ctypes.c_uint8 * nat.ROPE_MAX_PAIRS:
                ctypes.memset(ctypes.byref(getattr(a, name)), 7, nat.ROPE_MAX_PAIRS)
                want.append(bytes([7]) * nat.ROPE_MAX_PAIRS)
                continue
            arr = getattr(a, name)
            for k in range(typ._length_):
                i += 1
                arr[k] = i
                want.append(i)
        else:
            i += 1
            setattr(a, name, i)
            want.append(i)
    return a, want


@pytest.mark.parametrize("mirror,packer", [(nat.FdTablesArgs, "_TABLES_STRUCT"), (nat.FdRopeArgs, "_ROPE_STRUCT"),
                                           (nat.FdAttnArgs, "_ATTN_STRUCT")])
def test_packed_fields_land_where_the_mirror_has_them(mirror, packer):
    a, want = _numbered(mirror)
    assert bytes(a) == getattr(gpu_ops, packer).pack(*want)


def _rope():
    a = nat.FdRopeArgs()
    a.q = a.q_out = a.k = a.v = 4096
    a.positions, a.cos_sin, a.max_pos, a.slots = 4096, 4096, 10, None
    for f in ("q", "qo"):
        setattr(a, f + "_stride_t", 256), setattr(a, f + "_stride_h", 64)
    for f in ("k", "v"):
        setattr(a, f + "_stride_t", 128), setattr(a, f + "_stride_h", 64)
    a.num_tokens, a.num_heads, a.num_kv_heads, a.head_size, a.rot_dim = 3, 4, 2, 64, 64
    a.dtype, a.num_axes = 1, 1
    return a


@pytest.mark.parametrize("field,value,code,msg", [
    ("dtype", 9, 2, b"dtype"), ("num_tokens", -1, 1, b"shape"), ("num_heads", 0, 1, b"shape"),
    ("rot_dim", 63, 1, b"rot_dim"), ("rot_dim", 66, 1, b"rot_dim"), ("rot_dim", 0, 1, b"rot_dim"),
    ("num_axes", 0, 2, b"axes"), ("num_axes", 5, 2, b"axes"), ("q", None, 1, b"required"),
    ("positions", None, 1, b"required"), ("max_pos", 0, 1, b"required"), ("head_size", 68, 3, b"head_size"),
    ("k_stride_t", 132, 3, b"strides"), ("v", 4100, 3, b"aligned"), ("cos_sin", 4104, 3, b"aligned"),
    ("num_heads", 1 << 26, 2, b"too many"), ("slots", 4096, 1, b"block_size"),
])
def test_rope_rejects_bad_arguments(field, value, code, msg):
    a = _rope()
    setattr(a, field, value)
    assert nat.load().fd_rope_store_kv(ctypes.byref(a), None) == code
    assert msg in nat.load().fd_last_error_message()


def test_rope_rejects_an_axis_outside_the_positions():
    a = _rope()
    a.axis_of_pair[31] = 1
    assert nat.load().fd_rope_store_kv(ctypes.byref(a), None) == 1
    a = _rope()
    a.num_tokens = 0  # nothing to do
    assert nat.load().fd_rope_store_kv(ctypes.byref(a), None) == 0
    assert nat.load().fd_rope_store_kv(None, None) == 1


def _tables():
    a = nat.FdTablesArgs()
    for f in ("new_lens", "prior_lens", "block_table", "counts_in", "counts_out", "seq_lens", "query_start_loc",
              "slot_mapping", "positions", "header"):
        setattr(a, f, 4096)
    a.free_ids[0] = a.free_ids[1] = 4096
    a.free_cap[0] = a.free_cap[1] = 8
    a.bt_stride, a.bt_width, a.num_reqs, a.block_size, a.max_tokens = 8, 8, 4, 16, 32
    a.num_gpu_blocks, a.num_cpu_blocks = 8, 8
    return a


@pytest.mark.parametrize("field,value,code", [
    ("num_reqs", -1, 1), ("num_reqs", 8193, 2), ("max_tokens", -1, 1), ("max_tokens", (1 << 30) + 1, 2),
    ("block_size", 0, 1), ("bt_width", 0, 1), ("bt_stride", 7, 1), ("bt_width", 1 << 28, 1), ("counts_in", None, 1),
    ("header", None, 1), ("slot_mapping", None, 1), ("new_lens", None, 1), ("num_gpu_blocks", 1 << 31, 2),
])
def test_tables_reject_bad_arguments(field, value, code):
    a = _tables()
    setattr(a, field, value)
    assert nat.load().fd_extend_tables(ctypes.byref(a), None) == code
    a = _tables()
    a.free_ids[1] = None
    assert nat.load().fd_extend_tables(ctypes.byref(a), None) == 1
    a = _tables()
    a.bt_width, a.bt_stride = 1 << 28, 1 << 28
    assert nat.load().fd_extend_tables(ctypes.byref(a), None) == 2


def _attn(chunk=True):
    a = nat.FdAttnArgs()
    a.q = a.out = a.q_start = a.q_len = a.k_len = a.workspace = 4096
    a.workspace_bytes = 1 << 40
    a.q_stride_t, a.q_stride_h, a.out_stride_t, a.out_stride_h = 512, 64, 512, 64
    t = a.tier[0]
    t.k = t.v = 4096
    t.blk_stride, t.head_stride, t.tok_stride, t.num_blocks = 4096, 64, 256, 10
    if chunk:
        a.block_table, a.bt_stride, a.bt_width, a.block_size, a.tier_split = 4096, 4, 4, 16, 10
    else:
        a.k_start = 4096
    a.num_tokens, a.n, a.num_heads, a.num_kv_heads, a.head_size, a.scale, a.dtype = 4, 2, 8, 4, 64, 0.1, 0
    return a


@pytest.mark.parametrize("field,value,code,msg", [
    ("dtype", 5, 2, b"dtype"), ("n", -1, 1, b"negative"), ("n", 65536, 2, b"65535"), ("num_heads", 9, 1, b"multiple"),
    ("num_heads", 4 * 65, 2, b"group"), ("head_size", 264, 2, b"head_size"), ("head_size", 60, 3, b"head_size"),
    ("scale", 0.0, 1, b"scale"), ("scale", -1.0, 1, b"scale"), ("scale", float("nan"), 1, b"scale"),
    ("scale", float("inf"), 1, b"scale"), ("q", None, 1, b"required"), ("k_len", None, 1, b"required"),
    ("q", 4104, 3, b"aligned"), ("out_stride_h", 65, 3, b"aligned"), ("workspace", None, 4, b"workspace"),
    ("workspace_bytes", 16, 4, b"workspace"), ("workspace", 4100, 4, b"workspace"),
])
@pytest.mark.parametrize("chunk", [True, False])
def test_attention_rejects_bad_arguments(chunk, field, value, code, msg):
    lib = nat.load()
    a = _attn(chunk)
    setattr(a, field, value)
    name = "fd_chunk_attn" if chunk else "fd_cross_attn"
    assert getattr(lib, name)(ctypes.byref(a), None) == code
    text = lib.fd_last_error_message()
    assert msg in text and name.encode() in text


def test_attention_rejects_what_only_one_form_needs():
    lib = nat.load()
    for field in ("block_table", "bt_width", "block_size"):
        a = _attn()
        setattr(a, field, None if field == "block_table" else 0)
        assert lib.fd_chunk_attn(ctypes.byref(a), None) == 1
    a = _attn(False)
    a.k_start = None
    assert lib.fd_cross_attn(ctypes.byref(a), None) == 1
    a = _attn(False)
    a.tier[0].host_mapped = 1
    assert lib.fd_cross_attn(ctypes.byref(a), None) == 2
    a = _attn()
    a.tier[1].num_blocks = 3  # a tier without memory
    assert lib.fd_chunk_attn(ctypes.byref(a), None) == 1
    a = _attn()
    a.tier[0].tok_stride = 65
    assert lib.fd_chunk_attn(ctypes.byref(a), None) == 3
    for a in (_attn(), _attn(False)):
        a.n = 0
        assert lib.fd_chunk_attn(ctypes.byref(a), None) == 0
        assert lib.fd_cross_attn(None, None) == 1


def test_chunk_attention_rejects_a_negative_number_of_table_rows():
    a = _attn()
    a.bt_rows = -1
    assert nat.load().fd_chunk_attn(ctypes.byref(a), None) == 1
    assert b"bt_rows" in nat.load().fd_last_error_message()


def test_cross_attention_needs_pointers_of_states_that_are_there():
    lib = nat.load()
    for field in ("k", "v"):
        a = _attn(False)
        setattr(a.tier[0], field, None)
        assert lib.fd_cross_attn(ctypes.byref(a), None) == 1
        assert b"states" in lib.fd_last_error_message()
        a.tier[0].num_blocks, a.workspace = 0, None  # none are: on to the next check
        assert lib.fd_cross_attn(ctypes.byref(a), None) == 4


def test_workspace_grows_with_the_head_and_is_zero_for_no_head():
    lib = nat.load()
    a = _attn()
    small = lib.fd_attn_workspace_size(ctypes.byref(a))
    a.head_size = 128
    assert small > 0 and small % 256 == 0 and lib.fd_attn_workspace_size(ctypes.byref(a)) > small
    a.head_size = 0
    assert lib.fd_attn_workspace_size(ctypes.byref(a)) == 0


def test_axes_of_pairs():
    assert gpu_ops.rope_axes((2, 3)) == bytes([0, 0, 1, 1, 1])
    assert gpu_ops.rope_axes((4, 2, 1), True) == bytes([0, 1, 2, 0, 1, 0, 0])
    assert gpu_ops.rope_axes((0, 2)) == bytes([1, 1])
    for bad in ((), (0, 0), (1, 1, 1, 1, 1), (3, -1), (129,)):
        with pytest.raises(RuntimeError):
            gpu_ops.rope_axes(bad)


def test_bench_counts_a_cosine_and_a_sine_per_pair():
    """Bytes of the rotary bench: q, k, v in and out, and per token the angles of
    its pairs, each from one axis, three positions and a slot."""
    _, nbytes, _ = kernel_bench.case_rope_store_kv(torch.device("meta"))
    T, H, KVH, D = 16384, 32, 8, 128
    assert nbytes == 2 * T * (H + 2 * KVH) * D * 2 + T * (2 * (D // 2) * 4 + 3 * 8 + 8)


def test_front_end_refuses_host_tensors():
    q = torch.zeros(2, 4, 64, dtype=torch.float16)
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        gpu_ops.cross_attn(q, q, q, i, i, i, i, 1.0, q)
    with pytest.raises(RuntimeError, match="CUDA"):
        gpu_ops.rope_store_kv(q, q, q, i.long(), torch.zeros(4, 64), None, (None, None), 0)
    with pytest.raises(RuntimeError, match="CUDA"):
        gpu_ops.extend_tables(i, i, i.view(1, 1), gpu_ops.FreeBlocks(i, None, i), 1, 0, 16, max_tokens=4)
    with pytest.raises(RuntimeError, match="tier"):
        gpu_ops.chunk_attn(q, (None, None), 0, i.view(1, 1), i, i, i, 1.0, q)
