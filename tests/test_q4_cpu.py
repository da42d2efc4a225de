"""Host-only checks of 4-bit arenas and packed prompts: memory plan, argument
checks that need no device, the token strides the Python layer derives."""
import ctypes as C

import numpy as np
import pytest
import torch

import q4_reference as ref
from qx_b200 import MODEL_GRANITE, MODEL_QWEN3, Context, ExecutionPlan, KvArena, KvPrecision, QxError, _lib
from qx_b200.runtime import _token_stride, model_shape


def kv_bytes(desc):
    lib, kb, vb = _lib.load(), C.c_size_t(), C.c_size_t()
    return lib.qxc_kv_bytes(C.byref(desc), C.byref(kb), C.byref(vb)), kb.value, vb.value


@pytest.mark.parametrize("model,capacity", [(MODEL_GRANITE, 4096), (MODEL_QWEN3, 40960)])
def test_a_4bit_row_is_288_bytes(model, capacity):
    st, kb, vb = kv_bytes(_lib.KvDesc(model, 3, 5, capacity, _lib.Q4, _lib.Q4, 0))
    assert st == _lib.OK and kb == vb == 3 * 5 * capacity * 288
    lib, k2, v2 = _lib.load(), C.c_size_t(), C.c_size_t()
    d, pg = _lib.KvDesc(model, 3, 5, capacity, _lib.Q4, _lib.Q4, 0), _lib.KvPaging(64, 11)
    assert lib.qxc_kv_paged_bytes(C.byref(d), C.byref(pg), C.byref(k2), C.byref(v2)) == _lib.OK
    assert k2.value == v2.value == 3 * 11 * 64 * 288


def test_execution_plan_in_4_bits():
    plan = ExecutionPlan.granite_with_kv_precision(512, KvPrecision.Q4)
    assert plan.kv_bytes == 24 * 512 * 2 * 288


@pytest.mark.parametrize("desc,status", [
    (_lib.KvDesc(0, 1, 1, 16, _lib.Q4, _lib.F16, 0), _lib.ERR_UNSUPPORTED),
    (_lib.KvDesc(0, 1, 1, 16, _lib.F32, _lib.Q4, 0), _lib.ERR_UNSUPPORTED),
    (_lib.KvDesc(1, 1, 1, 16, _lib.BF16, _lib.Q4, 0), _lib.ERR_UNSUPPORTED),
    (_lib.KvDesc(1, 1, 1, 16, _lib.Q4, _lib.Q4, 64), _lib.ERR_UNSUPPORTED),
    (_lib.KvDesc(0, 1, 1, 4097, _lib.Q4, _lib.Q4, 0), _lib.ERR_INVALID_ARG),
    (_lib.KvDesc(1, 1, 1, 40961, _lib.Q4, _lib.Q4, 0), _lib.ERR_INVALID_ARG),
])
def test_descriptors_refused(desc, status):
    assert kv_bytes(desc)[0] == status


def test_null_arguments():
    lib = _lib.load()
    assert lib.qxc_kv_append(None, None, None) == _lib.ERR_INVALID_ARG
    assert lib.qxc_kv_read_rows(None, None, None) == _lib.ERR_INVALID_ARG
    assert lib.qxc_attend_packed(None, None) == _lib.ERR_INVALID_ARG
    assert lib.qxc_prefill_packed(None, None, None) == _lib.ERR_INVALID_ARG


def test_token_strides():
    x = torch.zeros(10, 24, 64)
    assert _token_stride(x, 24 * 64) == 24 * 64
    assert _token_stride(x[:, :16], 16 * 64) == 24 * 64  # part of a joint projection
    assert _token_stride(x[::2], 24 * 64) == 2 * 24 * 64
    assert _token_stride(x[:1, :16], 16 * 64) == 0       # one token: any stride
    assert _token_stride(None, 5) == 0 and _token_stride(4096, 5) == 0
    for bad, features in ((x[:, :, ::2], 24 * 32), (x.transpose(1, 2), 24 * 64), (x, 64),
                          (x[:1].expand(10, 24, 64), 24 * 64), (x[:, ::2], 12 * 64)):
        with pytest.raises(QxError):
            _token_stride(bad, features)


@pytest.mark.parametrize("model", [MODEL_GRANITE, MODEL_QWEN3])
@pytest.mark.parametrize("key", [True, False])
def test_the_stated_layout_uses_every_bit_once(model, key):
    """Each bit of the code bytes belongs to exactly one dim."""
    base = np.zeros((1, 288), np.uint8)
    owners = np.zeros((256, 8), np.int64)
    start, _ = ref.unpack_rows(model, base, key)
    for byte in range(256):
        for bit in range(8):
            raw = base.copy()
            raw[0, byte] ^= 1 << bit
            codes, _ = ref.unpack_rows(model, raw, key)
            changed = np.flatnonzero(codes != start)
            assert changed.size == 1
            owners[byte, bit] = changed[0]
    assert (np.bincount(owners.flatten(), minlength=512) == 4).all()


def test_reference_quantiser_rounds_ties_to_even_and_keeps_the_largest():
    x = np.zeros((1, 1, 64), np.float32)
    x[..., 0] = 7.0
    x[..., 1:5] = [0.5, 1.5, 2.5, -2.5]
    codes, scales = ref.quantise(x)
    assert scales[0, 0].tolist() == [1.0, 0.0]
    assert codes[0, 0, :5].tolist() == [14, 7, 9, 9, 5]
    assert (codes[0, 0, 32:] == 7).all()


class Calls:
    """A library that notes the calls it gets instead of making them."""

    def __init__(self):
        self.made = []

    def __getattr__(self, name):
        return lambda *args: self.made.append(name) or _lib.OK


def bare(model=MODEL_GRANITE, device=-1):
    """A context and a 4-bit arena without a GPU, whose device is the CPU."""
    ctx, arena = object.__new__(Context), object.__new__(KvArena)
    ctx.lib = arena.lib = Calls()
    ctx.handle = arena.handle = None
    ctx.device, arena.ctx, arena.model = device, ctx, model
    arena.layers, arena.sequences, arena.capacity = 1, 4, 64
    arena.key_dtype = arena.value_dtype = _lib.Q4
    arena.hq, arena.hkv, arena.d = model_shape(model)
    arena.row_shape = (288,)
    return ctx, arena


def refused(lib, call, status=_lib.ERR_INVALID_ARG, match=None):
    with pytest.raises(QxError, match=match) as e:
        call()
    assert e.value.status == status and not lib.made


@pytest.mark.parametrize("model", [MODEL_GRANITE, MODEL_QWEN3])
def test_outputs_must_be_dense(model):
    """A part of a joint projection may be an input; written as dense rows it would
    run over its neighbours."""
    ctx, arena = bare(model)
    lib, (hq, hkv, d) = arena.lib, model_shape(model)
    joint = torch.zeros(10, hq + 2 * hkv, d, dtype=torch.bfloat16)
    q, k, v = joint[:, :hq], joint[:, hq:hq + hkv], joint[:, hq + hkv:]
    dense = lambda x: torch.zeros(x.shape, dtype=x.dtype)  # noqa: E731
    append = lambda **kw: arena.append(q, k, v, [0], [10], in_dtype=_lib.BF16, **{"q_rot": dense(q), **kw})  # noqa: E731
    prefill = lambda out: arena.prefill_packed(q, k, v, out, [10])  # noqa: E731
    attend = lambda out: ctx.attend_packed(model, q, k, v, out, [10])  # noqa: E731
    read = lambda a, b: arena.read_rows(a, b, [0], [10], out_dtype=_lib.BF16)  # noqa: E731
    wide = torch.zeros(20, hq, d, dtype=torch.bfloat16)
    for call in (lambda: append(q_rot=q), lambda: append(k_rot=k), lambda: prefill(q), lambda: attend(q),
                 lambda: attend(wide[::2]), lambda: read(k, dense(v)), lambda: read(None, v)):
        refused(lib, call, match="dense")
    append(k_rot=dense(k))
    prefill(dense(q))
    attend(wide[10:])
    read(dense(k), dense(v))
    assert lib.made == ["qxc_kv_append", "qxc_prefill_packed", "qxc_attend_packed", "qxc_kv_read_rows"]


@pytest.mark.parametrize("model", [MODEL_GRANITE, MODEL_QWEN3])
def test_types_are_those_of_the_call(model):
    """A tensor of another type would be read or written past its end, or as other numbers."""
    ctx, arena = bare(model)
    lib, (hq, hkv, d) = arena.lib, model_shape(model)
    make = lambda h, t: torch.zeros(10, h, d, dtype=t)  # noqa: E731
    types = {_lib.F32: torch.float32, _lib.BF16: torch.bfloat16, _lib.F16: torch.float16}

    def append(t=torch.bfloat16, rot=torch.bfloat16, v=None, norm=None, **kw):
        arena.append(make(hq, t), make(hkv, t), make(hkv, v or t), [0], [10], in_dtype=_lib.BF16, q_rot=make(hq, rot),
                     k_rot=make(hkv, rot), k_norm=norm, **kw)
    read = lambda t, **kw: arena.read_rows(make(hkv, t), make(hkv, t), [0], [10], **kw)  # noqa: E731
    prefill = lambda t, o: arena.prefill_packed(make(hq, t), make(hkv, t), make(hkv, t), make(hq, o), [10])  # noqa: E731
    attend = lambda t, o: ctx.attend_packed(model, make(hq, t), make(hkv, t), make(hkv, t), make(hq, o), [10])  # noqa: E731
    b16, f16, f32 = torch.bfloat16, torch.float16, torch.float32
    bad = [lambda: append(f32), lambda: append(f16), lambda: append(torch.float64), lambda: append(v=f16),
           lambda: append(rot=f32), lambda: append(rot=torch.int8), lambda: read(b16), lambda: read(f32, out_dtype=_lib.F16),
           lambda: prefill(f32, b16), lambda: prefill(b16, f32), lambda: attend(f16, b16), lambda: attend(b16, f16)]
    if model == MODEL_QWEN3:
        bad += [lambda: append(norm=torch.zeros(d, dtype=b16)), lambda: append(norm=torch.zeros(2 * d)[::2]),
                lambda: append(norm=torch.zeros(d - 1))]
    for call in bad:
        refused(lib, call, match="type|dense|needed")
    for dt, t in types.items():
        read(t, out_dtype=dt)
    read(torch.int16, out_dtype=_lib.BF16)  # as KvArena.tensor shows 16-bit storage
    append()
    append(norm=torch.zeros(d))
    prefill(b16, b16)
    attend(b16, b16)
    assert len(lib.made) == 8


def test_tensors_are_on_the_context_device():
    """Host memory that the device cannot address, or another device's, would fault there."""
    ctx, arena = bare(device=0)
    q, k = torch.zeros(10, 16, 64, dtype=torch.bfloat16), torch.zeros(10, 8, 64, dtype=torch.bfloat16)
    raw = 1 << 20
    for call in (lambda: arena.append(None, k, raw, [0], [10], in_dtype=_lib.BF16),
                 lambda: arena.append(None, raw, raw, [0], [10], k_rot=k, in_dtype=_lib.BF16),
                 lambda: arena.append(None, k.float().numpy(), raw, [0], [10], in_dtype=_lib.F32),
                 lambda: arena.read_rows(k.float(), raw, [0], [10]), lambda: arena.read_rows(raw, k.float().numpy(), [0], [10]),
                 lambda: arena.prefill_packed(q, raw, raw, raw, [10]), lambda: arena.prefill_packed(raw, raw, raw, q, [10]),
                 lambda: ctx.attend_packed(MODEL_GRANITE, raw, raw, k, raw, [10])):
        refused(arena.lib, call, match="device|host")
    arena.read_rows(raw, raw, [0], [10])
    assert arena.lib.made == ["qxc_kv_read_rows"]


def test_a_tensor_without_tokens_is_refused():
    ctx, arena = bare()
    for x in (torch.zeros(()), torch.zeros(512)):
        refused(arena.lib, lambda: arena.append(None, x, x, [0], [1], in_dtype=_lib.F32))


def test_positions_and_sequences_of_a_decode():
    """Any iterable of numbers; as many sequences as positions are read by the library,
    so a list that is shorter is filled up and one that is longer is an error."""
    arena = bare()[1]
    args = lambda p, ids: arena._decode_args(1, 1, 1, 1, p, 0, 1, ids, 0, 0, 0, 0, 0, None, None, None)  # noqa: E731
    for p, ids in (([5, 7], [1, 0]), ((5, 7), np.array([1, 0])), (np.array([5.0, 7.0]), (x for x in (1, 0))),
                   ([5, 7.0], (x for x in (1.0, 0))),
                   (torch.tensor([5, 7]), torch.tensor([1.0, 0.0]))):
        pos, seq = args(p, ids)._keep
        assert list(pos) == [5, 7] and list(seq) == [1, 0]
    pos, seq = args([5, 7], [3])._keep
    assert len(seq) == 2 and list(seq) == [3, 0]
    with pytest.raises(IndexError):
        args([5, 7], [1, 0, 2])
    assert len(args([], None)._keep[0]) == 0 and len(args([], [])._keep[1]) == 0
    assert list(args([2 ** 31], None)._keep[0]) == [-2 ** 31]  # which the library refuses


def test_numbers_of_more_than_32_bits_are_refused():
    ctx, arena = bare()
    for big in (2 ** 31, -2 ** 31 - 1, 2 ** 40):
        for call in (lambda: arena.append(None, 1, 1, [big], [1]), lambda: arena.append(None, 1, 1, [0], [big]),
                     lambda: arena.append(None, 1, 1, [0], [1], seq_ids=[big]), lambda: arena.read_rows(1, 1, [big], [1]),
                     lambda: arena.prefill_packed(1, 1, 1, 1, [big]), lambda: ctx.attend_packed(0, 1, 1, 1, 1, [big])):
            refused(arena.lib, call)
    arena.append(None, 1, 1, np.array([0.0]), [1.0])
    assert arena.lib.made == ["qxc_kv_append"]


def test_raw_rows_written_to_a_4bit_arena():
    """Values are no rows: cut to bytes, the first 288 of 512 would be written."""
    arena = bare()[1]
    raw = np.zeros((3, 288), np.uint8)
    for k, v in ((np.zeros((3, 8, 64), np.float32), None), (raw[:, :287], None), (raw, raw[:2]), (raw, raw.astype(np.int32)),
                 (None, np.zeros((3, 8, 64), np.uint8))):
        refused(arena.lib, lambda: arena.write(0, 0, 0, k, v))
    arena.write(0, 0, 0, raw, None)
    arena.write(0, 0, 0, np.zeros((6, 288), np.uint8)[::2], raw)
    arena.write(0, 0, 0, torch.zeros(3, 288, dtype=torch.uint8), None)
    assert arena.lib.made == ["qxc_kv_write"] * 3


def test_types_that_a_call_refuses_reach_it():
    """The library says that a type is unsupported, not that a tensor has another."""
    ctx, arena = bare()
    q, k = torch.zeros(10, 16, 64, dtype=torch.bfloat16), torch.zeros(10, 8, 64, dtype=torch.bfloat16)
    for dt in (_lib.F32, _lib.Q4, 9):
        ctx.attend_packed(MODEL_GRANITE, q, k, k, torch.zeros_like(q), [10], dtype=dt)
        arena.prefill_packed(q, k, k, torch.zeros_like(q), [10], dtype=dt)
    for dt in (_lib.Q4, 9):
        arena.append(None, k, k, [0], [10], in_dtype=dt)
        arena.read_rows(k, k, [0], [10], out_dtype=dt)
    assert len(arena.lib.made) == 10


def test_a_seventh_without_a_division():
    """quantise8 makes top / 7 of a product with the rounded seventh and a correction by its
    residual: the correctly rounded quotient for every mantissa. (64 bits hold the residual,
    a few units of the quotient's last place, and the corrected sum exactly, so rounding
    that sum once to 32 bits is what a fused multiply-add does.)"""
    seventh = np.float32(1.0) / np.float32(7.0)
    for begin in range(0, 1 << 23, 1 << 21):
        top = (np.arange(begin, begin + (1 << 21), dtype=np.uint32) + np.uint32(0x3f800000)).view(np.float32)
        guess = top * seventh
        residual = top.astype(np.float64) - 7.0 * guess.astype(np.float64)
        # 7 times: half a unit of a guess in [1/4, 2/7), 2^-26, and top times the seventh's own error, 2 * 2^-27
        assert np.abs(residual).max() <= 7 * 2.0 ** -25
        got = (residual * np.float64(seventh) + guess.astype(np.float64)).astype(np.float32)
        assert np.array_equal(got, top / np.float32(7.0))
