"""4-bit arenas on the GPU: rows written and read back (codes compared
exactly), decode against attention in 64 bits over the stored values.

Tolerances. A weight p of the softmax is off by at most twice the largest
logit error (numerator and sum) plus 2^-20 for the hardware exponential and
the f32 sums along a split; with a 16-bit output the weights enter their
product with the values in fp16 (2^-11). An output is a mean of values under
those weights, so it is off by that relative error times the weighted mean of
|v|, plus half a step of its own type.

A weight times its row's scale s enters its product as one or two fp16 numbers,
the last of them off by at most half of fp16's smallest step, 2^-25, where the
row with the largest logit has weight 2^7 / (2 s_max) or more (the reference is
set from s_max rounded up to a power of two). Codes are at most 7, so N rows add
at most N * 7 * 2^-25 / (2^7 / (2 s_max)) = N * 2^-31 * 7 s_max, and 7 s_max is
the largest |v| a row can hold: N * 2^-31 * max |v| within its rounding. That is
what is left of dims whose heaviest rows hold zeros.
"""
import numpy as np
import pytest
import torch

import q4_reference as ref
from qx_b200 import (BF16, DECODE_NO_ADVANCE, F16, F32, MODEL_GRANITE, MODEL_QWEN3, Q4, Context, KvArena, QxError, _lib)
from qx_b200.runtime import model_shape

pytestmark = pytest.mark.gpu
MODELS = [MODEL_GRANITE, MODEL_QWEN3]


def tensor(rng, shape, dtype, scale=1.0):
    return (torch.from_numpy(rng.standard_normal(shape).astype(np.float32)) * scale).to(ref.TORCH[dtype]).cuda()


def host(x):
    return x.double().cpu().numpy()


def norms(rng, model):
    if model != MODEL_QWEN3:
        return None, None
    return tuple(torch.from_numpy((1.0 + 0.3 * rng.random(128)).astype(np.float32)).cuda() for _ in range(2))


def make_arena(ctx, model, rows, layers=1, page=0, capacity=None):
    cap = capacity or max(max(rows), 1)
    if not page:
        return KvArena(ctx, model, layers, len(rows), cap, Q4)
    pool = sum(-(-n // page) for n in rows) + 2
    return KvArena(ctx, model, layers, len(rows), cap, Q4, page_size=page, pool_pages=pool)


def stored(arena, seq, layer, begin, count):
    """(codes, scales) of keys and of values, from the raw rows."""
    return tuple(ref.unpack_rows(arena.model, raw, key) for raw, key in zip(arena.read(seq, layer, begin, count), (True, False)))


def granite_keys32(ctx, k, position):
    """The rotated f32 rows an f32 arena stores for keys k [tokens, 8, 64]."""
    n = k.shape[0]
    twin = KvArena(ctx, MODEL_GRANITE, 1, 1, position + n, F32)
    out = np.zeros((n, 8, 64), np.float32)
    zero, sink = torch.zeros(1024, device="cuda"), torch.zeros(1024, device="cuda")
    for i in range(n):
        twin.set_len(0, position + i)
        twin.decode(zero, k[i].float().contiguous(), k[i].float().contiguous(), sink, [position + i])
        out[i] = twin.read(0, 0, position + i, 1)[0][0]
    twin.close()
    return out


def keys32(ctx, model, k, position, norm):
    if model == MODEL_GRANITE:
        return granite_keys32(ctx, k, position)
    return ref.qwen_keys32(k.float().cpu().numpy(), range(position, position + k.shape[0]),
                           None if norm is None else norm.cpu().numpy())


@pytest.mark.parametrize("model", MODELS)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("starts,counts,page", [([0], [1], 0), ([700], [1], 64), ([0, 3, 63], [5, 0, 2], 64),
                                                ([1, 0, 60, 0], [1, 67, 9, 0], 128)])
def test_append_and_read_rows(gpu_ctx, model, dtype, starts, counts, page):
    rng = np.random.default_rng([model, dtype, sum(counts), page])
    hq, hkv, d = model_shape(model)
    layers, total = 2, sum(counts)
    arena = make_arena(gpu_ctx, model, [s + c for s, c in zip(starts, counts)], layers, page)
    for i, s in enumerate(starts):
        arena.set_len(i, s)
    qw, kw = norms(rng, model)
    q, k, v = (tensor(rng, (total, layers, h, d), dtype, 2.0) for h in (hq, hkv, hkv))
    q_rot = torch.zeros(total, layers, hq, d, device="cuda")
    k_rot = torch.zeros(total, layers, hkv, d, device="cuda")
    arena.append(q, k, v, starts, counts, in_dtype=dtype, q_rot=q_rot, k_rot=k_rot, rot_dtype=F32, q_norm=qw, k_norm=kw)
    gpu_ctx.sync()
    assert [arena.len(i) for i in range(len(counts))] == [s + c for s, c in zip(starts, counts)]
    outs = {dt: [torch.zeros(total, layers, hkv, d, device="cuda", dtype=ref.TORCH[dt]) for _ in range(2)]
            for dt in (F32, BF16, F16)}
    for dt, (ko, vo) in outs.items():
        arena.read_rows(ko, vo, starts, counts, out_dtype=dt)
    gpu_ctx.sync()
    at = 0
    for i, (s, c) in enumerate(zip(starts, counts)):
        if not c:
            continue
        part = slice(at, at + c)
        at += c
        pos = np.arange(s, s + c)
        for l in range(layers):
            for x, rot, w in ((q, q_rot, qw), (k, k_rot, kw)):
                want = ref.rotate64(model, host(x[part, l]), pos, None if w is None else host(w))
                half = d // 2
                size = np.hypot(want[..., :half], want[..., half:])
                # about eight roundings of a pair (norm, weight, cos, sin, two products, their sum)
                assert ref.close(host(rot[part, l]), want, 8 * 2.0 ** -24 * np.concatenate([size, size], -1) + 1e-30) <= 1
            (kc, ks), (vc, vs) = stored(arena, i, l, s, c)
            want_k = ref.quantise(keys32(gpu_ctx, model, k[part, l], s, kw))
            want_v = ref.quantise(v[part, l].float().cpu().numpy())
            assert np.array_equal(ks, want_k[1]) and np.array_equal(kc, want_k[0])
            assert np.array_equal(vs, want_v[1]) and np.array_equal(vc, want_v[0])
            for dt, (ko, vo) in outs.items():
                for got, cs in ((ko, (kc, ks)), (vo, (vc, vs))):
                    want = torch.from_numpy(ref.values(*cs)).to(ref.TORCH[dt])
                    assert torch.equal(got[part, l].cpu(), want)
    arena.close()


@pytest.mark.parametrize("model", MODELS)
def test_append_leaves_other_rows(gpu_ctx, model):
    rng = np.random.default_rng(5)
    hq, hkv, d = model_shape(model)
    arena = KvArena(gpu_ctx, model, 3, 3, 20, Q4)
    for s in range(3):
        for l in range(3):
            for key in (True, False):
                arena.tensor(s, l, key).fill_(0xA5)
    arena.set_len(2, 4)
    k, v = (tensor(rng, (3, 1, hkv, d), BF16) for _ in range(2))
    arena.append(None, k, v, [4], [3], seq_ids=[2], layer_begin=1, layer_count=1, in_dtype=BF16, flags=DECODE_NO_ADVANCE)
    gpu_ctx.sync()
    assert arena.len(2) == 4
    for s in range(3):
        for l in range(3):
            for key in (True, False):
                changed = (arena.tensor(s, l, key) != 0xA5).any(1).nonzero().flatten().tolist()
                assert changed == ([4, 5, 6] if (s, l) == (2, 1) else [])
    arena.close()


@pytest.mark.parametrize("model", MODELS)
def test_append_strided_and_unaligned_inputs(gpu_ctx, model):
    rng = np.random.default_rng(6)
    hq, hkv, d = model_shape(model)
    n = 19
    joint = tensor(rng, (n, hq + 2 * hkv, d), BF16)
    parts = [joint[:, :hq], joint[:, hq:hq + hkv], joint[:, hq + hkv:]]
    shifted = []
    for x in parts:  # the same values one element past a 16-byte boundary, odd token stride
        flat = torch.zeros(n, x[0].numel() + 3, device="cuda", dtype=torch.bfloat16)
        view = flat.flatten()[1:]
        view = torch.as_strided(view, (n, x[0].numel()), (x[0].numel() + 3, 1))
        view.copy_(x.flatten(1))
        shifted.append(view)
    got = []
    for q, k, v in ([x.contiguous() for x in parts], parts, shifted):
        arena = KvArena(gpu_ctx, model, 1, 1, n, Q4)
        rot = torch.zeros(n * hq * d + 8, device="cuda", dtype=torch.float16)
        rot = rot[1:1 + n * hq * d] if q is shifted[0] else rot[:n * hq * d]
        arena.append(q, k, v, [0], [n], in_dtype=BF16, q_rot=rot, rot_dtype=F16)
        gpu_ctx.sync()
        got.append((rot.clone(), *(x.copy() for x in arena.read(0, 0, 0, n))))
        arena.close()
    for other in got[1:]:
        assert torch.equal(got[0][0], other[0])
        assert np.array_equal(got[0][1], other[1]) and np.array_equal(got[0][2], other[2])


@pytest.mark.parametrize("model", MODELS)
def test_rows_at_the_ends_of_the_scale(gpu_ctx, model):
    """Zero groups, groups whose scale is subnormal or rounds to zero, groups of one large value."""
    hkv, d = model_shape(model)[1:]
    top = np.array([0.0, 1e-9, 3e-7, 6e-7, 1e-5, 1.0, 4e5, 7 * 65504.0], np.float32)
    v = np.linspace(-1, 1, 32, dtype=np.float32) * top[:, None]
    v = np.resize(v, (2, hkv, d)).astype(np.float32)
    arena = KvArena(gpu_ctx, model, 1, 1, 2, Q4)
    arena.append(None, torch.zeros(2, hkv, d, device="cuda"), torch.from_numpy(v).cuda(), [0], [2], in_dtype=F32)
    gpu_ctx.sync()
    (kc, ks), (vc, vs) = stored(arena, 0, 0, 0, 2)
    assert (kc == 7).all() and (ks == 0).all()
    want = ref.quantise(v)
    assert np.array_equal(vs, want[1]) and np.array_equal(vc, want[0])
    arena.close()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), 1e6])
@pytest.mark.parametrize("side", ["k", "v"])
def test_values_without_a_scale_are_reported(gpu_ctx, bad, side):
    arena = KvArena(gpu_ctx, MODEL_GRANITE, 1, 1, 4, Q4)
    x = {"k": torch.ones(1, 8, 64, device="cuda"), "v": torch.ones(1, 8, 64, device="cuda")}
    x[side][0, 3, 37] = bad
    arena.append(None, x["k"], x["v"], [0], [1], in_dtype=F32)
    with pytest.raises(QxError) as e:
        gpu_ctx.sync()
    assert e.value.status == _lib.ERR_NONFINITE
    arena.append(None, torch.ones(1, 8, 64, device="cuda"), torch.ones(1, 8, 64, device="cuda"), [1], [1], in_dtype=F32)
    gpu_ctx.sync()
    arena.close()


def test_read_rows_in_any_order(gpu_ctx):
    rng = np.random.default_rng(8)
    hkv, d = model_shape(MODEL_QWEN3)[1:]
    arena = make_arena(gpu_ctx, MODEL_QWEN3, [130, 70], page=64)
    k, v = (tensor(rng, (200, hkv, d), F16) for _ in range(2))
    arena.append(None, k, v, [0, 0], [130, 70], in_dtype=F16)
    every = [torch.zeros(200, hkv, d, device="cuda") for _ in range(2)]
    arena.read_rows(*every, [0, 0], [130, 70])
    begins, counts, ids = [60, 1, 0, 129, 64], [9, 3, 0, 1, 6], [0, 1, 1, 0, 1]
    got = [torch.full((sum(counts) + 1, hkv, d), 9.0, device="cuda") for _ in range(2)]
    arena.read_rows(*got, begins, counts, seq_ids=ids)
    only = torch.zeros(3, hkv, d, device="cuda")
    arena.read_rows(None, only, [1], [3], seq_ids=[1])
    gpu_ctx.sync()
    rows = torch.cat([torch.arange(b, b + c) + (130 if i else 0) for b, c, i in zip(begins, counts, ids)]).cuda()
    for g, e in zip(got, every):
        assert torch.equal(g[:-1], e[rows]) and (g[-1] == 9.0).all()
    assert torch.equal(only, every[1][131:134])
    arena.close()


# ---- decode ------------------------------------------------------------------------
def fill(ctx, arena, rng, rows, kw=None, scale=1.0, dtype=BF16):
    """Cached rows of every sequence and layer; returns their stored values."""
    hkv, d = arena.hkv, arena.d
    for l in range(arena.layers):
        for i in range(len(rows)):
            arena.set_len(i, 0)
        if sum(rows):
            k = tensor(rng, (sum(rows), hkv, d), dtype, scale)
            k[:, :, 5] *= 4.0
            v = tensor(rng, (sum(rows), hkv, d), dtype)
            arena.append(None, k, v, [0] * len(rows), rows, layer_begin=l, layer_count=1, in_dtype=dtype, k_norm=kw)
    for i, n in enumerate(rows):
        arena.set_len(i, n)
    ctx.sync()


def check_decode(ctx, arena, q, k, v, out, positions, out_dtype, qw=None, kw=None, ids=None, layer_begin=0):
    """`out` of a decode against 64 bits over what the arena holds now."""
    model = arena.model
    for i, pos in enumerate(positions):
        seq = ids[i] if ids else i
        for l in range(q.shape[1]):
            (kc, ks), (vc, vs) = stored(arena, seq, layer_begin + l, 0, pos + 1)
            new_v = ref.quantise(v[i, l].float().cpu().numpy()[None])
            assert np.array_equal(vc[-1:], new_v[0]) and np.array_equal(vs[-1:], new_v[1])
            keys, vals = ref.values(kc, ks), ref.values(vc, vs)
            qr = ref.rotate64(model, host(q[i, l])[None], [pos], None if qw is None else host(qw))[0]
            want, mean = ref.attend64(model, qr, keys, vals)
            # a dot product of D terms in chains of at most 64, the query's own rotation (8) and split (4)
            weights = 2 * ref.logit_error(model, qr, keys, 76) + 2.0 ** -20 + (0 if out_dtype == F32 else 2.0 ** -11)
            floor = (pos + 1) * 2.0 ** -31 * 7 * vs.astype(np.float64).max()
            floor += 2.0 ** -25 if out_dtype == F16 else 1e-30  # half of an fp16 output's smallest step
            tol = ref.HALF_STEP[out_dtype] * np.abs(want) + weights * mean + floor
            assert ref.close(host(out[i, l]), want, tol) <= 1, (i, l, pos)


def run_decode(ctx, arena, rng, positions, dtype, out_dtype, qw=None, kw=None, ids=None, layer_begin=0, layer_count=None,
               split=0, q_scale=1.0, check=True):
    layers = arena.layers - layer_begin if layer_count is None else layer_count
    n, hq, hkv, d = len(positions), arena.hq, arena.hkv, arena.d
    q, k, v = tensor(rng, (n, layers, hq, d), dtype, q_scale), tensor(rng, (n, layers, hkv, d), dtype), tensor(rng, (n, layers, hkv, d), dtype)
    out = torch.full((n, layers, hq, d), 7.0, device="cuda", dtype=ref.TORCH[out_dtype])
    arena.decode(q, k, v, out, positions, layer_begin=layer_begin, layer_count=layers, seq_ids=ids, q_dtype=dtype,
                 in_dtype=dtype, out_dtype=out_dtype, split=split, q_norm=qw, k_norm=kw)
    ctx.sync()
    if check:
        check_decode(ctx, arena, q, k, v, out, positions, out_dtype, qw, kw, ids, layer_begin)
    return out


@pytest.mark.parametrize("model", MODELS)
@pytest.mark.parametrize("rows", [0, 1, 15, 30, 31, 32, 33, 63, 64, 65, 127, 128, 511, 1000])
@pytest.mark.parametrize("dtype,out_dtype", [(F32, F32), (BF16, BF16), (F16, F16)])
def test_decode_lengths(gpu_ctx, model, rows, dtype, out_dtype):
    rng = np.random.default_rng([model, rows, dtype])
    qw, kw = norms(rng, model)
    arena = make_arena(gpu_ctx, model, [rows], capacity=rows + 2)
    fill(gpu_ctx, arena, rng, [rows], kw)
    run_decode(gpu_ctx, arena, rng, [rows], dtype, out_dtype, qw, kw)
    assert arena.len(0) == rows + 1
    arena.close()


@pytest.mark.parametrize("model,longest", [(MODEL_GRANITE, 4095), (MODEL_QWEN3, 9001)])
@pytest.mark.parametrize("split", [0, 64, 192, 1024])
@pytest.mark.parametrize("out_dtype", [F32, BF16])
def test_decode_splits(gpu_ctx, model, longest, split, out_dtype):
    rng = np.random.default_rng([model, split])
    qw, kw = norms(rng, model)
    arena = make_arena(gpu_ctx, model, [longest], capacity=longest + 1)
    fill(gpu_ctx, arena, rng, [longest], kw)
    run_decode(gpu_ctx, arena, rng, [longest], BF16, out_dtype, qw, kw, split=split)
    arena.close()


@pytest.mark.parametrize("model", MODELS)
@pytest.mark.parametrize("page", [0, 64, 256])
def test_decode_ragged_batch_over_steps(gpu_ctx, model, page):
    """Uneven sequences, some of them in the call, pages that end inside a tile, three steps in a row."""
    rng = np.random.default_rng([model, page])
    qw, kw = norms(rng, model)
    rows = [0, 63, 64, 700, 1, 255, 129]
    arena = make_arena(gpu_ctx, model, [n + 4 for n in rows], layers=3, page=page)
    fill(gpu_ctx, arena, rng, rows, kw)
    ids = [6, 0, 3, 2, 4, 1]
    for step in range(3):
        run_decode(gpu_ctx, arena, rng, [rows[i] + step for i in ids], BF16, F32, qw, kw, ids=ids)
    assert [arena.len(i) for i in range(7)] == [n + (3 if i in ids else 0) for i, n in enumerate(rows)]
    arena.close()


def test_decode_layer_range(gpu_ctx):
    rng = np.random.default_rng(9)
    arena = make_arena(gpu_ctx, MODEL_GRANITE, [100, 3], layers=4, capacity=128)
    fill(gpu_ctx, arena, rng, [100, 3])
    before = [x.copy() for x in arena.read(0, 0, 0, 128)]
    run_decode(gpu_ctx, arena, rng, [100, 3], F32, F32, layer_begin=1, layer_count=2)
    assert all(np.array_equal(a, b) for a, b in zip(before, arena.read(0, 0, 0, 128)))
    arena.close()


@pytest.mark.parametrize("model", MODELS)
def test_decode_more_sequences_than_a_launch_holds(gpu_ctx, model):
    rng = np.random.default_rng(10)
    rows = [int(x) for x in rng.integers(0, 90, 421)]
    arena = make_arena(gpu_ctx, model, [n + 1 for n in rows], page=64)
    fill(gpu_ctx, arena, rng, rows)
    run_decode(gpu_ctx, arena, rng, rows, BF16, BF16)
    arena.close()


@pytest.mark.parametrize("model", MODELS)
@pytest.mark.parametrize("out_dtype", [F32, BF16])
def test_decode_does_not_read_past_the_new_token(gpu_ctx, model, out_dtype):
    """Every byte behind the last row is 0xFF: NaN scales, codes of 15."""
    rng = np.random.default_rng(11)
    rows = [5, 64, 99]
    arena = make_arena(gpu_ctx, model, [n + 1 for n in rows], capacity=200)
    for s in range(3):
        for key in (True, False):
            arena.tensor(s, 0, key).fill_(0xFF)
    fill(gpu_ctx, arena, rng, rows)
    run_decode(gpu_ctx, arena, rng, rows, BF16, out_dtype)
    arena.close()


@pytest.mark.parametrize("model", MODELS)
@pytest.mark.parametrize("v_scale", [2.0 ** -20, 2.0 ** -9, 1.0, 2.0 ** 14])
@pytest.mark.parametrize("out_dtype", [F32, BF16])
def test_decode_value_ranges(gpu_ctx, model, v_scale, out_dtype):
    """Values far from 1, and in the last rows 1000 times larger (or smaller) than in the first."""
    rng = np.random.default_rng(12)
    hkv, d = model_shape(model)[1:]
    rows = 333
    arena = make_arena(gpu_ctx, model, [rows + 1])
    k, v = tensor(rng, (rows, hkv, d), F32), tensor(rng, (rows, hkv, d), F32, v_scale)
    v[200:] *= 2.0 ** -10 if v_scale > 1 else 2.0 ** 10
    v[:, 0, :32] = 0.0
    arena.append(None, k, v, [0], [rows], in_dtype=F32)
    q, k1, v1 = tensor(rng, (1, 1, arena.hq, d), F32), tensor(rng, (1, 1, hkv, d), F32), tensor(rng, (1, 1, hkv, d), F32, v_scale)
    out = torch.zeros(1, 1, arena.hq, d, device="cuda", dtype=ref.TORCH[out_dtype])
    arena.decode(q, k1, v1, out, [rows], q_dtype=F32, in_dtype=F32, out_dtype=out_dtype)
    gpu_ctx.sync()
    check_decode(gpu_ctx, arena, q, k1, v1, out, [rows], out_dtype)
    arena.close()


@pytest.mark.parametrize("q_scale", [0.0, 1e-6, 40.0])
def test_decode_flat_and_peaked_scores(gpu_ctx, q_scale):
    rng = np.random.default_rng(13)
    arena = make_arena(gpu_ctx, MODEL_GRANITE, [301])
    fill(gpu_ctx, arena, rng, [300], scale=3.0)
    run_decode(gpu_ctx, arena, rng, [300], F32, F32, q_scale=q_scale)
    arena.close()


def test_decode_mixed_input_types_and_rotated_query(gpu_ctx):
    rng = np.random.default_rng(14)
    arena = make_arena(gpu_ctx, MODEL_GRANITE, [71])
    fill(gpu_ctx, arena, rng, [70])
    q, k, v = tensor(rng, (1, 1, 16, 64), F32), tensor(rng, (1, 1, 8, 64), F16), tensor(rng, (1, 1, 8, 64), F16)
    out, rot = torch.zeros(1, 1, 16, 64, device="cuda"), torch.zeros(1, 1, 16, 64, device="cuda")
    arena.decode(q, k, v, out, [70], q_dtype=F32, in_dtype=F16, q_rot_out=rot)
    gpu_ctx.sync()
    check_decode(gpu_ctx, arena, q, k, v, out, [70], F32)
    want = ref.rotate64(MODEL_GRANITE, host(q[0]), [70])
    size = np.hypot(want[..., :32], want[..., 32:])
    assert ref.close(host(rot[0]), want, 8 * 2.0 ** -24 * np.concatenate([size, size], -1)) <= 1
    arena.close()


def test_decode_host_buffers(gpu_ctx):
    rng = np.random.default_rng(15)
    arena = make_arena(gpu_ctx, MODEL_GRANITE, [41])
    fill(gpu_ctx, arena, rng, [40])
    q, k, v = (rng.standard_normal((1, n)).astype(np.float32) for n in (1024, 512, 512))
    out = arena.decode_host(q, k, v, [40])
    as_dev = [torch.from_numpy(x).cuda().view(1, 1, -1, 64) for x in (q, k, v)]
    check_decode(gpu_ctx, arena, *as_dev, torch.from_numpy(out).view(1, 1, 16, 64), [40], F32)
    arena.close()


def test_unaligned_decode_inputs(gpu_ctx):
    rng = np.random.default_rng(16)
    arena = make_arena(gpu_ctx, MODEL_QWEN3, [41])
    fill(gpu_ctx, arena, rng, [40])
    q, k, v = (torch.zeros(n * 128 + 1, device="cuda", dtype=torch.bfloat16)[1:] for n in (32, 4, 4))
    for x in (q, k, v):
        x.copy_(tensor(rng, x.shape, BF16))
    out = torch.zeros(4097, device="cuda", dtype=torch.bfloat16)[1:]
    arena.decode(q, k, v, out, [40], out_dtype=BF16)
    gpu_ctx.sync()
    check_decode(gpu_ctx, arena, *(x.view(1, 1, -1, 128) for x in (q, k, v, out)), [40], BF16)
    arena.close()


def test_decode_captured_and_replayed(gpu_ctx):
    """A captured step replays with new inputs; what the arena holds changes under it in between."""
    rng = np.random.default_rng(17)
    arena = make_arena(gpu_ctx, MODEL_QWEN3, [3001, 41], page=64)
    fill(gpu_ctx, arena, rng, [3000, 40])
    shape = lambda h: (2, 1, h, 128)  # noqa: E731
    q, k, v = (tensor(rng, shape(h), BF16) for h in (32, 4, 4))
    out = torch.zeros(*shape(32), device="cuda")
    step = lambda: arena.decode(q, k, v, out, [3000, 40], out_dtype=F32, flags=DECODE_NO_ADVANCE)  # noqa: E731
    old = gpu_ctx.stream
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        gpu_ctx.set_stream(stream)
        step()  # sizes the workspaces
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
        for _ in range(3):
            for x in (q, k, v):
                x.copy_(tensor(rng, x.shape, BF16))
            out.zero_()
            graph.replay()
            stream.synchronize()
            check_decode(gpu_ctx, arena, q, k, v, out, [3000, 40], F32)
    gpu_ctx.set_stream(old)
    arena.close()


def test_a_captured_step_outlives_a_larger_one():
    """A captured decode keeps its workspace when a later call needs a larger
    one; a call that needs a larger one cannot be captured."""
    rng = np.random.default_rng(19)
    ctx = Context(0)
    stream = torch.cuda.Stream()
    arena = make_arena(ctx, MODEL_GRANITE, [701] * 30, layers=3)
    fill(ctx, arena, rng, [700] * 30)
    q, k, v = (tensor(rng, (1, 3, h, 64), BF16) for h in (16, 8, 8))
    out = torch.zeros(1, 3, 16, 64, device="cuda")
    small = lambda: arena.decode(q, k, v, out, [700], q_dtype=BF16, in_dtype=BF16, flags=DECODE_NO_ADVANCE)  # noqa: E731
    lq, lk, lv = (tensor(rng, (30, 3, h, 64), BF16) for h in (16, 8, 8))
    lout = torch.zeros(30, 3, 16, 64, device="cuda")
    large = lambda: arena.decode(lq, lk, lv, lout, [700] * 30, q_dtype=BF16, in_dtype=BF16, flags=DECODE_NO_ADVANCE)  # noqa: E731
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        ctx.set_stream(stream)
        small()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            small()
        with pytest.raises(QxError) as e:
            with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=stream):
                small()  # a graph with no node cannot be made
                large()
        assert e.value.status == _lib.ERR_UNSUPPORTED
        for _ in range(2):
            large()
            stream.synchronize()
            check_decode(ctx, arena, lq, lk, lv, lout, [700] * 30, F32)
            out.zero_()
            graph.replay()
            stream.synchronize()
            check_decode(ctx, arena, q, k, v, out, [700], F32)
    ctx.sync()
    arena.close()
    ctx.close()


def test_two_contexts_at_once(gpu_ctx):
    """Contexts of their own stream and workspaces do not wait for each other."""
    rng = np.random.default_rng(24)
    both = [(Context(0), m) for m in MODELS]
    work = []
    for ctx, model in both:
        arena = make_arena(ctx, model, [2001, 301])
        fill(ctx, arena, rng, [2000, 300])
        q, k, v = (tensor(rng, (2, 1, h, arena.d), BF16) for h in (arena.hq, arena.hkv, arena.hkv))
        work.append((ctx, arena, q, k, v, torch.zeros(2, 1, arena.hq, arena.d, device="cuda")))
    torch.cuda.synchronize()
    for _ in range(20):
        for ctx, arena, q, k, v, out in work:
            arena.decode(q, k, v, out, [2000, 300], q_dtype=BF16, in_dtype=BF16, flags=DECODE_NO_ADVANCE)
    for ctx, arena, q, k, v, out in work:
        ctx.sync()
        check_decode(ctx, arena, q, k, v, out, [2000, 300], F32)
        arena.close()
        ctx.close()


def test_offsets_past_32_bits(gpu_ctx):
    """The last rows of an arena whose keys alone pass 2^32 bytes: written, read
    back and attended, its other cells left as they were."""
    rng = np.random.default_rng(25)
    cap, layers, seqs = 40960, 40, 10
    arena = KvArena(gpu_ctx, MODEL_QWEN3, layers, seqs, cap, Q4)
    assert cap * layers * seqs * 288 > 2 ** 32
    k, v = (tensor(rng, (cap - 1, 4, 128), BF16) for _ in range(2))
    arena.append(None, k, v, [0], [cap - 1], seq_ids=[seqs - 1], layer_begin=layers - 1, layer_count=1, in_dtype=BF16)
    gpu_ctx.sync()
    keys, values = (torch.zeros(3, 1, 4, 128, device="cuda") for _ in range(2))
    arena.read_rows(keys, values, [cap - 4], [3], seq_ids=[seqs - 1], layer_begin=layers - 1, layer_count=1)
    gpu_ctx.sync()
    codes, scales = ref.quantise(v[-3:].float().cpu().numpy())
    assert np.array_equal(host(values)[:, 0], ref.values(codes, scales))
    run_decode(gpu_ctx, arena, rng, [cap - 1], BF16, F32, ids=[seqs - 1], layer_begin=layers - 1, layer_count=1)
    arena.close()


@pytest.mark.parametrize("model", MODELS)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rotation_in_place(gpu_ctx, model, dtype):
    rng = np.random.default_rng([model, dtype, 26])
    arena = make_arena(gpu_ctx, model, [130, 130])
    qw, kw = norms(rng, model)
    q, k, v = (tensor(rng, (130, h, arena.d), dtype) for h in (arena.hq, arena.hkv, arena.hkv))
    got = []
    for seq, (a, b) in enumerate(((torch.zeros_like(q), torch.zeros_like(k)), (q, k))):
        arena.append(q, k, v, [0], [130], seq_ids=[seq], q_rot=a, k_rot=b, in_dtype=dtype, rot_dtype=dtype, q_norm=qw,
                     k_norm=kw)
        gpu_ctx.sync()
        got.append((a, b, *arena.read(seq, 0, 0, 130)))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    assert all(np.array_equal(x, y) for x, y in zip(got[0][2:], got[1][2:]))
    arena.close()


def test_q4_layer_runs_on_a_4bit_arena(gpu_ctx):
    """qxc_attention_layer decodes whatever arena it is given."""
    rng = np.random.default_rng(18)
    from qx_b200 import Q4Weights

    def weights(rows):
        codes = torch.from_numpy(rng.integers(0, 256, (rows, 32, 16), dtype=np.uint8)).cuda()
        scales = torch.full((rows, 32), 0.01, dtype=torch.float16).cuda()
        return Q4Weights(codes, scales, rows, 1024)
    w = [weights(n) for n in (1024, 512, 512, 1024)]
    x, norm = tensor(rng, (1024,), F32), torch.ones(1024, device="cuda")
    got = []
    for dt in (F32, Q4):
        arena = KvArena(gpu_ctx, MODEL_GRANITE, 1, 1, 8, dt)
        att, out = torch.zeros(1024, device="cuda"), torch.zeros(1024, device="cuda")
        arena.attention_layer(x, out, norm, *w, position=0, attention_out=att)
        gpu_ctx.sync()
        got.append(att)
        arena.close()
    # one position: the attention is its value row, off by at most half a code step (a fourteenth of the group's largest)
    step = got[0].view(-1, 32).abs().amax(1, keepdim=True) / 14 * (1 + 2.0 ** -9)
    assert ((got[0] - got[1]).view(-1, 32).abs() <= step).all()


@pytest.mark.parametrize("page", [0, 64])
def test_a_stack_of_layers_on_a_4bit_arena(gpu_ctx, page):
    """qxc_attention_stack is its layers one after another, bit for bit."""
    rng = np.random.default_rng([27, page])
    from qx_b200 import Q4Weights

    def weights(rows):
        codes = torch.from_numpy(rng.integers(0, 256, (rows, 32, 16), dtype=np.uint8)).cuda()
        return Q4Weights(codes, torch.full((rows, 32), 0.01, dtype=torch.float16).cuda(), rows, 1024)
    layers = [{"norm": torch.ones(1024, device="cuda"), **{n: weights(r) for n, r in zip("qkvo", (1024, 512, 512, 1024))}}
              for _ in range(3)]
    stack, chain = (KvArena(gpu_ctx, MODEL_GRANITE, 3, 1, 70, Q4, page_size=page, pool_pages=2 if page else 0) for _ in range(2))
    for position in range(66):
        x = tensor(rng, (1024,), F32)
        out, y = torch.zeros(1024, device="cuda"), x.clone()
        stack.attention_stack(x, out, layers, position)
        for i, w in enumerate(layers):
            z = torch.zeros(1024, device="cuda")
            chain.attention_layer(y, z, w["norm"], w["q"], w["k"], w["v"], w["o"], position=position, layer=i,
                                  flags=DECODE_NO_ADVANCE if i < 2 else 0)
            y = z
        gpu_ctx.sync()
        assert torch.equal(out, y) and torch.isfinite(y).all()
    assert stack.len(0) == chain.len(0) == 66
    for i in range(3):
        assert all(np.array_equal(a, b) for a, b in zip(stack.read(0, i, 0, 66), chain.read(0, i, 0, 66)))
    stack.close()
    chain.close()


def test_refusals(gpu_ctx):
    arena = KvArena(gpu_ctx, MODEL_GRANITE, 2, 2, 64, Q4)
    plain = KvArena(gpu_ctx, MODEL_GRANITE, 1, 1, 64, F32)
    k = torch.zeros(70, 2, 8, 64, device="cuda")
    q = torch.zeros(70, 2, 16, 64, device="cuda")

    def refused(status, call):
        launches = gpu_ctx.launch_count
        with pytest.raises(QxError) as e:
            call()
        assert e.value.status == status and gpu_ctx.launch_count == launches and str(e.value)
    bad, pos, unsupported = _lib.ERR_INVALID_ARG, _lib.ERR_POSITION, _lib.ERR_UNSUPPORTED
    app = lambda p, c, a=arena, **kw: a.append(None, k, k, p, c, in_dtype=F32, **kw)  # noqa: E731
    one = k[:, :1]
    refused(unsupported, lambda: plain.append(None, one, one, [0], [1], in_dtype=F32))
    refused(pos, lambda: app([1], [1]))
    refused(pos, lambda: app([0], [65]))
    refused(pos, lambda: app([0], [2 ** 31 - 1]))
    refused(bad, lambda: app([0], [-1]))
    refused(bad, lambda: app([0, 0], [1, 1], seq_ids=[1, 1]))
    refused(bad, lambda: app([0], [1], seq_ids=[2]))
    refused(bad, lambda: app([0], [1], layer_begin=1, layer_count=2))
    refused(bad, lambda: app([0], [1], layer_begin=-1, layer_count=2))
    refused(bad, lambda: app([], []))
    refused(bad, lambda: app([0, 0], [1]))
    refused(bad, lambda: arena.append(None, k, None, [0], [1], in_dtype=F32))
    refused(bad, lambda: arena.append(q, k, k, [0], [1], in_dtype=F32))
    refused(bad, lambda: arena.append(None, k, k, [0], [1], in_dtype=Q4))
    refused(bad, lambda: arena.append(None, k[:, :, ::2], k, [0], [1], in_dtype=F32))
    refused(unsupported, lambda: plain.read_rows(k, k, [0], [1]))
    refused(pos, lambda: arena.read_rows(k, k, [60], [5]))
    refused(bad, lambda: arena.read_rows(k, k, [-1], [1]))
    refused(bad, lambda: arena.read_rows(None, None, [0], [1]))
    refused(bad, lambda: arena.read_rows(k, k, [0], [1], out_dtype=Q4))
    out = torch.zeros(16 * 64, device="cuda")
    dec = lambda **kw: arena.decode(out, out, out, out, kw.pop("p", [0]), layer_count=1, **kw)  # noqa: E731
    refused(pos, lambda: dec(p=[1]))
    refused(bad, lambda: dec(split=32))
    refused(bad, lambda: dec(split=-64))
    refused(bad, lambda: dec(in_dtype=Q4))
    refused(bad, lambda: dec(p=[0, 0], seq_ids=[0, 0]))
    refused(unsupported, lambda: dec(flags=_lib.DECODE_PINNED_EXP))
    refused(unsupported, lambda: arena.decode_verify(q, k, k, q, 0, 2))
    refused(unsupported, lambda: arena.decode_partials(out, out, out, out, 0, True))
    refused(unsupported, lambda: arena.prefill(q, k, k, q, 4))
    app([0], [3])
    refused(unsupported, lambda: arena.slot_hashes(out, 0, 1, 0, 1))
    gpu_ctx.sync()
    paged = KvArena(gpu_ctx, MODEL_GRANITE, 1, 2, 256, Q4, page_size=64, pool_pages=2)
    refused(_lib.ERR_OUT_OF_MEMORY, lambda: paged.append(None, one, one, [0, 0], [65, 5], in_dtype=F32))
    assert paged.page_stats() == (0, 2)
    refused(bad, lambda: paged.read_rows(k, k, [0], [1]))
    for a in (arena, plain, paged):
        a.close()


# ---- steps that follow one another ---------------------------------------------------
@pytest.mark.parametrize("model", MODELS)
@pytest.mark.parametrize("seqs,layers,rows", [(1, 24, 64), (112, 2, 64), (128, 3, 128), (148, 6, 64), (213, 2, 100), (5, 4, 700)])
def test_steps_without_a_synchronisation_between_them(gpu_ctx, model, seqs, layers, rows):
    """Steps with different inputs, one behind another on the stream, give what each
    gives alone. In most of these shapes the borders of the cells are borders of CTAs,
    so the grid that joins parts finds none."""
    rng = np.random.default_rng([model, seqs, layers, rows])
    steps, at = 6, [rows - 1] * seqs
    arena = make_arena(gpu_ctx, model, [rows] * seqs, layers)
    fill(gpu_ctx, arena, rng, at)
    ins = [[tensor(rng, (seqs, layers, h, arena.d), BF16) for h in (arena.hq, arena.hkv, arena.hkv)] for _ in range(steps)]
    outs = [[torch.zeros(seqs, layers, arena.hq, arena.d, device="cuda", dtype=torch.bfloat16) for _ in range(steps)]
            for _ in range(2)]
    gpu_ctx.sync()
    for i, alone in enumerate((False, True)):
        for _ in range(1 if alone else 4):
            for (q, k, v), out in zip(ins, outs[i]):
                arena.decode(q, k, v, out, at, q_dtype=BF16, in_dtype=BF16, out_dtype=BF16, flags=DECODE_NO_ADVANCE)
                if alone:
                    gpu_ctx.sync()
        gpu_ctx.sync()
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    some = sorted({0, seqs // 2, seqs - 1})
    q, k, v = ([x[some] for x in ins[-1]])
    check_decode(gpu_ctx, arena, q, k, v, outs[0][-1][some], [rows - 1] * len(some), BF16, ids=some)
    arena.close()


def test_an_append_right_behind_a_step(gpu_ctx):
    """An append into sequences that were reset right after a decode was enqueued does
    not reach the rows which that decode still reads."""
    rng = np.random.default_rng(31)
    seqs, layers, rows = 112, 2, 64
    arena = make_arena(gpu_ctx, MODEL_GRANITE, [rows] * seqs, layers)
    q, k, v = (tensor(rng, (seqs, layers, h, 64), BF16) for h in (16, 8, 8))
    ak, av = (tensor(rng, (seqs * (rows - 1), layers, 8, 64), BF16) for _ in range(2))
    other = tensor(rng, (seqs * (rows - 1), layers, 8, 64), BF16, 3.0)
    outs = []
    for behind in (True, False):
        out = torch.zeros(seqs, layers, 16, 64, device="cuda", dtype=torch.bfloat16)
        for _ in range(8):
            arena.reset(-1)
            arena.append(None, ak, av, [0] * seqs, [rows - 1] * seqs, in_dtype=BF16)
            arena.decode(q, k, v, out, [rows - 1] * seqs, q_dtype=BF16, in_dtype=BF16, out_dtype=BF16)
            if behind:
                arena.reset(-1)
                arena.append(None, other, other, [0] * seqs, [rows - 1] * seqs, in_dtype=BF16)
            gpu_ctx.sync()
            outs.append(out.clone())
    assert all(torch.equal(outs[-1], o) for o in outs)
    arena.close()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size", [1e17, 1e20, 1e30, 3e37])
def test_norms_of_the_largest_queries_and_keys(gpu_ctx, dtype, size):
    """Elements whose squares pass f32: the norm brings any of them back to size 1."""
    rng = np.random.default_rng([dtype, int(np.log10(size))])
    arena = make_arena(gpu_ctx, MODEL_QWEN3, [41])
    q, k = (tensor(rng, (40, 1, h, 128), dtype) for h in (32, 4))
    q[3:, 0, 5:9] *= size
    q[::2, 0, 20, 77] = size
    k[:, 0, 1] *= size
    v = tensor(rng, (40, 1, 4, 128), dtype)
    rot, keys = torch.zeros(40, 1, 32, 128, device="cuda"), torch.zeros(40, 1, 4, 128, device="cuda")
    arena.append(q, k, v, [0], [40], in_dtype=dtype, q_rot=rot, k_rot=keys, rot_dtype=F32)
    gpu_ctx.sync()
    for x, got in ((q, rot), (k, keys)):
        want = ref.rotate64(MODEL_QWEN3, host(x[:, 0]), range(40))
        pair = np.hypot(want[..., :64], want[..., 64:])
        # as in test_append_and_read_rows; the reciprocal of a root beyond 2^126 has fewer
        # bits: half a step of 2^-149 of at least 2^-128
        assert ref.close(host(got[:, 0]), want, (8 * 2.0 ** -24 + 2.0 ** -22) * np.concatenate([pair, pair], -1) + 1e-30) <= 1
    dq = tensor(rng, (1, 1, 32, 128), dtype)
    dq[0, 0, 4:7] *= size
    dk, dv = tensor(rng, (1, 1, 4, 128), dtype, size), tensor(rng, (1, 1, 4, 128), dtype)
    out, turned = torch.zeros(1, 1, 32, 128, device="cuda"), torch.zeros(1, 1, 32, 128, device="cuda")
    arena.decode(dq, dk, dv, out, [40], q_dtype=dtype, in_dtype=dtype, q_rot_out=turned)
    gpu_ctx.sync()
    want = ref.rotate64(MODEL_QWEN3, host(dq[0]), [40])
    pair = np.hypot(want[..., :64], want[..., 64:])
    assert ref.close(host(turned[0]), want, (8 * 2.0 ** -24 + 2.0 ** -22) * np.concatenate([pair, pair], -1) + 1e-30) <= 1
    if size < 1e37:  # (check_decode knows of eight roundings of a query)
        check_decode(gpu_ctx, arena, dq, dk, dv, out, [40], F32)
    arena.close()


def refused_capture(ctx, status, *calls):
    """The last of `calls` is refused under capture."""
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    ctx.set_stream(stream)
    with torch.cuda.stream(stream), pytest.raises(QxError) as e:
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=stream):
            for call in calls:
                launches = ctx.launch_count
                call()
    assert e.value.status == status
    ctx.set_stream(None)
    return ctx.launch_count - launches


def test_a_refused_capture_of_many_sequences_holds_none_of_its_launches():
    """The last of three launches is the one whose workspace is too small."""
    rng = np.random.default_rng(34)
    ctx = Context(0)
    rows = [1] * 400 + [2000] * 30
    arena = make_arena(ctx, MODEL_GRANITE, [n + 1 for n in rows], page=64)
    fill(ctx, arena, rng, rows)
    q, k, v = (tensor(rng, (430, 1, h, 64), BF16) for h in (16, 8, 8))
    out = torch.zeros(430, 1, 16, 64, device="cuda")
    torch.cuda.synchronize()
    go = lambda n: arena.decode(q, k, v, out, rows[:n], q_dtype=BF16, in_dtype=BF16, flags=DECODE_NO_ADVANCE)  # noqa: E731
    go(400)
    ctx.sync()
    assert refused_capture(ctx, _lib.ERR_UNSUPPORTED, lambda: go(200), lambda: go(430)) == 0
    go(430)
    ctx.sync()
    some = [0, 199, 200, 399, 400, 429]
    check_decode(ctx, arena, q[some], k[some], v[some], out[some], [rows[i] for i in some], F32, ids=some)
    arena.close()
    ctx.close()


def test_a_refused_capture_maps_no_page():
    """A mapping that is captured and thrown away with the graph would leave the device without it."""
    rng = np.random.default_rng(35)
    ctx = Context(0)
    arena = KvArena(ctx, MODEL_QWEN3, 1, 2, 200, Q4, page_size=64, pool_pages=6)
    fill(ctx, arena, rng, [64, 64])
    q, k, v = (tensor(rng, (2, 1, h, 128), BF16) for h in (32, 4, 4))
    out = torch.zeros(2, 1, 32, 128, device="cuda")
    torch.cuda.synchronize()
    go = lambda n: arena.decode(q, k, v, out, [64] * n, out_dtype=F32)  # noqa: E731
    kv = [torch.zeros(1, 1, 4, 128, device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    refused_capture(ctx, _lib.ERR_UNSUPPORTED, lambda: arena.read_rows(*kv, [0], [1]), lambda: go(2))
    assert arena.page_stats() == (2, 4) and [arena.len(i) for i in range(2)] == [64, 64]
    go(2)
    ctx.sync()
    assert arena.page_stats() == (4, 2)
    check_decode(ctx, arena, q, k, v, out, [64, 64], F32)
    arena.close()
    ctx.close()


def test_an_allocation_that_fails_is_reported_once():
    """An arena larger than the GPU is refused; the arenas, pages and steps after it are not."""
    rng = np.random.default_rng(37)
    for model in MODELS:
        ctx = Context(0)
        for page in (0, 64):
            with pytest.raises(QxError) as e:
                KvArena(ctx, model, 48, 4000, 4096, Q4, page_size=page, pool_pages=200000)
            assert e.value.status == _lib.ERR_OUT_OF_MEMORY
            arena = KvArena(ctx, model, 1, 1, 70, Q4, page_size=page, pool_pages=2)
            fill(ctx, arena, rng, [66])
            run_decode(ctx, arena, rng, [66], BF16, F32)
            arena.close()
        ctx.close()


@pytest.mark.parametrize("model", MODELS)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("q_scale,loud", [(1.0, 1.0), (1.0, 30.0), (40.0, 1.0)])
def test_decode_peaked_scores_into_bf16(gpu_ctx, model, dtype, q_scale, loud):
    """For a bf16 output a query head's elements are rounded to multiples of its largest /
    16128, off by half of that: a logit by up to that times the sum of a key's |elements|,
    twice in a weight (its own and the sum's)."""
    rng = np.random.default_rng([model, dtype, 39])
    arena = make_arena(gpu_ctx, model, [301])
    fill(gpu_ctx, arena, rng, [300], scale=3.0)
    hq, hkv, d = model_shape(model)
    q, k, v = (tensor(rng, (1, 1, h, d), dtype) for h in (hq, hkv, hkv))
    q[..., 9] *= loud
    qw = torch.full((128,), q_scale, device="cuda") if model == MODEL_QWEN3 else None  # (its norm undoes q's own scale)
    q = q if model == MODEL_QWEN3 else q * q_scale
    out = torch.zeros(1, 1, hq, d, device="cuda", dtype=torch.bfloat16)
    arena.decode(q, k, v, out, [300], q_dtype=dtype, in_dtype=dtype, out_dtype=BF16, q_norm=qw)
    gpu_ctx.sync()
    (kc, ks), (vc, vs) = stored(arena, 0, 0, 0, 301)
    keys, vals = ref.values(kc, ks), ref.values(vc, vs)
    qr = ref.rotate64(model, host(q[0, 0])[None], [300], None if qw is None else host(qw))[0]
    want, mean = ref.attend64(model, qr, keys, vals)
    size = np.repeat(np.abs(keys).sum(-1).max(0), hq // hkv)  # of each query head's keys
    logit = np.abs(qr).max(-1) / 16128 / 2 * size * ref.SCALE[model] + ref.logit_error(model, qr, keys, 76)
    weights = np.expm1(2 * logit)[:, None] + 2.0 ** -20 + 2.0 ** -11
    tol = ref.HALF_STEP[BF16] * np.abs(want) + weights * mean + 301 * 2.0 ** -31 * 7 * vs.astype(np.float64).max()
    assert ref.close(host(out[0, 0]), want, tol) <= 1
    arena.close()


@pytest.mark.parametrize("model", MODELS)
@pytest.mark.parametrize("parts", [2, 7, 8, 9, 12, 16, 17, 18, 33])
@pytest.mark.parametrize("out_dtype", [F32, BF16])
def test_decode_joins_any_number_of_parts(gpu_ctx, model, parts, out_dtype):
    """On both sides of the numbers from which on several threads share an output's parts."""
    rng = np.random.default_rng([model, parts])
    rows = [64 * parts - 3, 64 * (parts - 1), 1, 64 * parts - 64 + 5]
    arena = make_arena(gpu_ctx, model, [n + 1 for n in rows], layers=2)
    fill(gpu_ctx, arena, rng, rows)
    run_decode(gpu_ctx, arena, rng, rows, BF16, out_dtype, split=64)
    arena.close()


def test_overlapping_tensors_are_refused(gpu_ctx):
    """Warps read inputs and write outputs in any order, so only an output in its own
    input's place is written by the warp that has read it."""
    arena = KvArena(gpu_ctx, MODEL_GRANITE, 1, 1, 64, Q4)
    joint = torch.zeros(10, 32, 64, device="cuda", dtype=torch.bfloat16)
    q, k, v = joint[:, :16], joint[:, 16:24], joint[:, 24:]
    dq, dk, dv = (x.clone() for x in (q, k, v))
    flat = joint.view(-1)
    inside, behind = flat[:10 * 1024].view(10, 16, 64), torch.zeros(10, 16, 64, device="cuda", dtype=torch.bfloat16)

    def refused(call):
        launches = gpu_ctx.launch_count
        with pytest.raises(QxError, match="overlap") as e:
            call()
        assert e.value.status == _lib.ERR_INVALID_ARG and gpu_ctx.launch_count == launches
    append = lambda q, k, v, **kw: arena.append(q, k, v, [0], [10], in_dtype=BF16, flags=DECODE_NO_ADVANCE, **kw)  # noqa: E731
    refused(lambda: append(q, k, v, q_rot=inside))
    refused(lambda: append(None, k, v, k_rot=flat[-5120:].view(10, 8, 64)))
    refused(lambda: append(dq, dk, dv, q_rot=dq.view(-1), k_rot=dv))
    refused(lambda: append(dq, dk, dv, q_rot=behind, k_rot=behind.view(-1)[5120:]))
    refused(lambda: append(dq, dk, dk.view(10, 8, 64), q_rot=behind, k_rot=dk))
    refused(lambda: append(dq, dk, dv, q_rot=dq.data_ptr(), rot_dtype=F32))
    refused(lambda: arena.read_rows(dk, dk, [0], [10], out_dtype=BF16))
    refused(lambda: arena.read_rows(behind.view(-1)[8:], behind, [0], [9], out_dtype=BF16))
    refused(lambda: gpu_ctx.attend_packed(MODEL_GRANITE, q, k, v, inside, [10]))
    refused(lambda: gpu_ctx.attend_packed(MODEL_GRANITE, dq, dk, dv, dq, [10]))
    refused(lambda: arena.prefill_packed(dq, dk, behind[:, :8], behind, [10]))
    append(dq, dk, dv, q_rot=dq, k_rot=dk)
    append(q, k, v, q_rot=dq, k_rot=dk)
    arena.read_rows(dk, dv, [0], [10], out_dtype=BF16)
    arena.read_rows(flat[:512], flat[512:], [0], [1], out_dtype=BF16)
    gpu_ctx.attend_packed(MODEL_GRANITE, q, k, v, behind, [10])
    gpu_ctx.attend_packed(MODEL_GRANITE, behind[:4], k, v, behind[4:], [4])
    arena.prefill_packed(dq, dk, dv, dq, [10])  # its rotated queries are copies
    gpu_ctx.sync()
    arena.close()


def test_pages_mapped_by_a_capture_that_is_thrown_away(gpu_ctx):
    """The device gets their table entries from the next call that runs, also one that only reads."""
    rng = np.random.default_rng(41)
    hkv, d = model_shape(MODEL_QWEN3)[1:]
    old, stream = gpu_ctx.stream, torch.cuda.Stream()
    k, v = (tensor(rng, (300, hkv, d), BF16) for _ in range(2))
    torch.cuda.synchronize()
    graphs = []  # kept: one that goes while another is captured ends that capture
    for first in ("append", "read", "decode", "capture"):
        graphs += [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
        arena = KvArena(gpu_ctx, MODEL_QWEN3, 1, 2, 400, Q4, page_size=64, pool_pages=14)
        append = lambda seq, flags=0: arena.append(None, k, v, [0], [300], seq_ids=[seq], in_dtype=BF16, flags=flags)  # noqa: E731
        gpu_ctx.set_stream(stream)
        with torch.cuda.stream(stream), pytest.raises(KeyError):
            with torch.cuda.graph(graphs[-1], stream=stream):
                append(1, DECODE_NO_ADVANCE)
                append(1, DECODE_NO_ADVANCE)
                raise KeyError
        assert arena.page_stats(1)[0] == 5
        if first == "read":
            got = [torch.ones(300, hkv, d, device="cuda") for _ in range(2)]
            stream.wait_stream(torch.cuda.default_stream())
            arena.read_rows(*got, [0], [300], seq_ids=[1])
            gpu_ctx.sync()
            assert not got[0].any() and not got[1].any()  # rows that were never written
        elif first == "decode":
            arena.set_len(1, 300)
            run_decode(gpu_ctx, arena, rng, [300], BF16, F32, ids=[1], check=False)
            arena.set_len(1, 0)
        if first == "capture":
            with torch.cuda.stream(stream):
                with torch.cuda.graph(graphs[-2], stream=stream):
                    append(1)
                graphs[-2].replay()
        else:
            append(1)
        append(0)
        gpu_ctx.sync()
        gpu_ctx.set_stream(old)
        want = ref.quantise(v.float().cpu().numpy())
        rows = [stored(arena, seq, 0, 0, 300) for seq in range(2)]
        for (kc, ks), (vc, vs) in rows:
            assert np.array_equal(vc, want[0]) and np.array_equal(vs, want[1])
        assert np.array_equal(rows[0][0][0], rows[1][0][0]) and arena.page_stats() == (10, 4)
        torch.cuda.synchronize()
        run_decode(gpu_ctx, arena, rng, [300, 300], BF16, F32)
        arena.close()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_head_is_normed_alike_whatever_the_others_hold(gpu_ctx, dtype):
    """Heads whose squares pass f32 are normed another way; the heads beside them are not."""
    rng = np.random.default_rng([dtype, 42])
    q, k, v = (tensor(rng, (64, 1, h, 128), dtype) for h in (32, 4, 4))
    big = q.clone()
    big[:, :, ::3] *= 1e25
    rest = [h for h in range(32) if h % 3]
    got = []
    for x in (q, big):
        arena = make_arena(gpu_ctx, MODEL_QWEN3, [65])
        rot, turned, out = (torch.zeros(n, 1, 32, 128, device="cuda") for n in (64, 1, 1))
        arena.append(x, k, v, [0], [64], in_dtype=dtype, q_rot=rot, rot_dtype=F32)
        arena.decode(x[:1], k[:1], v[:1], out, [64], q_dtype=dtype, in_dtype=dtype, q_rot_out=turned)
        gpu_ctx.sync()
        got.append([y[:, :, rest] for y in (rot, turned, out)])
        arena.close()
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize("model", MODELS)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("page", [0, 64])
def test_a_step_writes_the_rows_that_an_append_writes(gpu_ctx, model, dtype, page):
    """Raw rows of keys and values, bit for bit, and the same outputs and rows from inputs
    that start one element past a 16-byte boundary."""
    rng = np.random.default_rng([model, dtype, page, 43])
    hq, hkv, d = model_shape(model)
    qw, kw = norms(rng, model)
    rows = [0, 1, 63, 64, 200]
    arenas = [make_arena(gpu_ctx, model, [n + 1 for n in rows], layers=2, page=page) for _ in range(3)]
    q, k, v = (tensor(rng, (5, 2, h, d), dtype, 2.0) for h in (hq, hkv, hkv))
    old = [tensor(rng, (sum(rows), 2, hkv, d), dtype) for _ in range(2)]
    for a in arenas:
        a.append(None, *old, [0] * 5, rows, in_dtype=dtype, k_norm=kw)
    shifted = []
    for x in (q, k, v):
        flat = torch.zeros(x.numel() + 1, device="cuda", dtype=x.dtype)[1:]
        shifted.append(flat.copy_(x.flatten()).view(x.shape))
    outs = [torch.zeros(5, 2, hq, d, device="cuda") for _ in range(2)]
    for a, ins, out in zip(arenas, ((q, k, v), shifted), outs):
        a.decode(*ins, out, rows, q_dtype=dtype, in_dtype=dtype, q_norm=qw, k_norm=kw)
    arenas[2].append(None, k, v, rows, [1] * 5, in_dtype=dtype, k_norm=kw)
    gpu_ctx.sync()
    assert torch.equal(*outs)
    for i, n in enumerate(rows):
        for l in range(2):
            raw = [a.read(i, l, 0, n + 1) for a in arenas]
            for other in raw[1:]:
                assert all(np.array_equal(x, y) for x, y in zip(raw[0], other))
    for a in arenas:
        a.close()


@pytest.mark.parametrize("model,capacity", [(MODEL_GRANITE, 4096), (MODEL_QWEN3, 40960)])
def test_a_prompt_that_fills_its_sequence(gpu_ctx, model, capacity):
    """The longest positions of a model: written by a prefill, read back, and then full."""
    rng = np.random.default_rng([model, 44])
    hq, hkv, d = model_shape(model)
    arena = KvArena(gpu_ctx, model, 1, 1, capacity, Q4)
    q, k, v = (tensor(rng, (capacity, h, d), BF16) for h in (hq, hkv, hkv))
    out = torch.zeros(capacity, hq, d, device="cuda", dtype=torch.bfloat16)
    arena.prefill_packed(q, k, v, out, [capacity])
    keys, values = (torch.zeros(2, hkv, d, device="cuda") for _ in range(2))
    arena.read_rows(keys, values, [capacity - 2], [2])
    gpu_ctx.sync()
    assert arena.len(0) == capacity and torch.isfinite(out).all()
    want = ref.quantise(keys32(gpu_ctx, model, k[-2:], capacity - 2, None))
    assert np.array_equal(host(keys), ref.values(*want))
    want = ref.quantise(v[-2:].float().cpu().numpy())
    assert np.array_equal(host(values), ref.values(*want))
    one = [x[:1, None] for x in (q, k, v)]
    for call in (lambda: arena.decode(*one, out[:1], [capacity], q_dtype=BF16, in_dtype=BF16, out_dtype=BF16),
                 lambda: arena.append(None, *one[1:], [capacity], [1], in_dtype=BF16)):
        with pytest.raises(QxError) as e:
            call()
        assert e.value.status == _lib.ERR_POSITION
    arena.close()
