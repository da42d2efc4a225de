"""Packed prompts: causal attention against 64 bits, and prompt, cache and
decode as a serving step runs them.

Tolerances. The weights of a key tile are rounded to the input type for their
product with the values (half a step of it) and come from a base-2 exponential
with a relative error of at most 2^-13; a logit error enters twice and sum); the sum of a row's weights in f32 adds its length in roundings. fp16
has a smallest step, 2^-24: a weight is off by up to half of it where the key
that set the reference has weight 1 (so the weights' sum is 1 or more), N of
them times max |v|, and so is the output.
"""
import numpy as np
import pytest
import torch

import q4_reference as ref
from qx_b200 import BF16, F16, F32, MODEL_GRANITE, MODEL_QWEN3, Q4, Context, KvArena, QxError, _lib
from qx_b200.runtime import model_shape
from test_q4_gpu import check_decode, host, norms, stored, tensor

pytestmark = pytest.mark.gpu
MODELS = [MODEL_GRANITE, MODEL_QWEN3]


def inputs(rng, model, total, dtype, fused=False):
    hq, hkv, d = model_shape(model)
    if fused:
        joint = tensor(rng, (total, hq + 2 * hkv, d), dtype, 1.2)
        return joint[:, :hq], joint[:, hq:hq + hkv], joint[:, hq + hkv:]
    return tensor(rng, (total, hq, d), dtype, 1.5), tensor(rng, (total, hkv, d), dtype), tensor(rng, (total, hkv, d), dtype)


def check(model, q, k, v, out, lengths, dtype, heads=None):
    """Every row of `out` against 64 bits (on the GPU: prompts may be long)."""
    hq, hkv, d = model_shape(model)
    begin = 0
    for n in lengths:
        rows = slice(begin, begin + n)
        begin += n
        for h in heads or range(hq):
            kd, vd = k[rows, h * hkv // hq].double(), v[rows, h * hkv // hq].double()
            qd = q[rows, h].double()
            for at in range(0, n, 1024):
                part = qd[at:at + 1024]
                seen = at + part.shape[0]
                later = torch.arange(seen, device="cuda") > torch.arange(at, seen, device="cuda")[:, None]
                logits = (part @ kd[:seen].T * ref.SCALE[model]).masked_fill(later, -torch.inf)
                p = torch.softmax(logits, -1)
                want, mean = p @ vd[:seen], p @ vd[:seen].abs()
                # products are exact in f32, D of them summed in f32
                size = (part.abs() @ kd[:seen].abs().T).masked_fill(later, 0).amax(-1, keepdim=True) * ref.SCALE[model]
                rel = 2 * size * (d + 2) * 2.0 ** -24 + ref.HALF_STEP[dtype] + 2.0 ** -13 + seen * 2.0 ** -24
                floor = 2.0 ** -25 * (1 + seen * float(vd[:seen].abs().max())) if dtype == F16 else 1e-30
                tol = ref.HALF_STEP[dtype] * want.abs() + rel * mean + floor
                got = out[rows, h][at:seen].double()
                assert torch.isfinite(got).all()
                assert float(((got - want).abs() / tol).max()) <= 1, (n, h, at)


def attend(ctx, model, q, k, v, lengths, dtype, extra=0):
    hq, _, d = model_shape(model)
    out = torch.full((q.shape[0] + extra, hq, d), 5.0, device="cuda", dtype=ref.TORCH[dtype])
    ctx.attend_packed(model, q, k, v, out, lengths, dtype=dtype)
    ctx.sync()
    assert (out[sum(lengths):] == 5.0).all()
    return out


@pytest.mark.parametrize("model", MODELS)
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 400])
def test_one_prompt(gpu_ctx, model, n):
    rng = np.random.default_rng([model, n])
    for dtype in (BF16, F16):
        q, k, v = inputs(rng, model, n, dtype)
        check(model, q, k, v, attend(gpu_ctx, model, q, k, v, [n], dtype, 2), [n], dtype)


@pytest.mark.parametrize("model", MODELS)
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lengths", [[3, 0, 1, 130, 64, 0, 257, 1], [0, 0, 5], [100, 28, 128, 128], [1] * 40])
def test_packed_prompts(gpu_ctx, model, dtype, lengths):
    rng = np.random.default_rng([model, dtype, len(lengths)])
    q, k, v = inputs(rng, model, sum(lengths), dtype, fused=True)
    check(model, q, k, v, attend(gpu_ctx, model, q, k, v, lengths, dtype, 3), lengths, dtype)


@pytest.mark.parametrize("model", MODELS)
def test_more_prompts_than_a_launch_holds(gpu_ctx, model):
    rng = np.random.default_rng(3)
    lengths = [int(x) for x in rng.integers(0, 9, 450)]
    q, k, v = inputs(rng, model, sum(lengths), BF16)
    check(model, q, k, v, attend(gpu_ctx, model, q, k, v, lengths, BF16), lengths, BF16)


def test_no_tokens(gpu_ctx):
    launches = gpu_ctx.launch_count
    out = torch.full((2, 16, 64), 5.0, device="cuda", dtype=torch.bfloat16)
    gpu_ctx.attend_packed(MODEL_GRANITE, None, None, None, out, [0, 0])
    gpu_ctx.sync()
    assert gpu_ctx.launch_count == launches and (out == 5.0).all()


@pytest.mark.parametrize("model", MODELS)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_a_row_does_not_attend_does_not_reach_it(gpu_ctx, model, bad):
    """A bad key and value at token 90 of prompt 1: rows of other prompts and
    the 90 rows before it are as without it, the rows from it on are not finite."""
    rng = np.random.default_rng(4)
    lengths = [70, 200, 50]
    q, k, v = inputs(rng, model, sum(lengths), BF16)
    clean = attend(gpu_ctx, model, q, k, v, lengths, BF16)
    at = lengths[0] + 90
    rest = torch.cat([torch.arange(at), torch.arange(270, 320)]).cuda()
    for side in (k, v):
        keep = side[at].clone()
        side[at] = bad
        out = torch.zeros_like(clean)
        gpu_ctx.attend_packed(model, q, k, v, out, lengths, dtype=BF16)
        with pytest.raises(QxError) as e:
            gpu_ctx.sync()
        assert e.value.status == _lib.ERR_NONFINITE
        side[at] = keep
        if side is v:
            assert not torch.isfinite(out[at:270]).any()
        check(model, q[:at], k[:at], v[:at], out[:at], [70, 90], BF16)
        check(model, q[270:], k[270:], v[270:], out[270:], [50], BF16)
        assert torch.equal(out[270:], clean[270:]) and torch.equal(out[:70], clean[:70]) and rest.numel() == at + 50


@pytest.mark.parametrize("model", MODELS)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_a_bad_value_reaches_its_own_dim_only(gpu_ctx, model, dtype):
    """Values of two dims are bad from one token on: the rows from it on have
    these dims not finite and the others right, the rows before it all right."""
    rng = np.random.default_rng([model, dtype, 20])
    n = 300
    q, k, v = inputs(rng, model, n, dtype)
    bad = {130: (5, float("nan")), 201: (40, float("-inf"))}
    clean = v.clone()
    for at, (dim, x) in bad.items():
        v[at:, :, dim] = x
    out = torch.zeros_like(q)
    gpu_ctx.attend_packed(model, q, k, v, out, [n], dtype=dtype)
    with pytest.raises(QxError) as e:
        gpu_ctx.sync()
    assert e.value.status == _lib.ERR_NONFINITE
    for at, (dim, _) in bad.items():
        assert not torch.isfinite(out[at:, :, dim]).any()
        out[at:, :, dim] = 0.0
        clean[at:, :, dim] = 0.0
    # a zeroed value from a row on is a zeroed output from it on, the rows before are as they were
    for at, (dim, _) in bad.items():
        check_dim(model, q, k, v, out, at, dim, dtype)
    assert torch.isfinite(out).all()
    keep = [d for d in range(q.shape[2]) if d not in (5, 40)]
    check_columns(model, q, k, clean, out, n, dtype, keep)


def check_columns(model, q, k, v, out, n, dtype, columns):
    """As check() for one prompt, some of its output dims."""
    only = torch.zeros(v.shape[2], device="cuda", dtype=v.dtype)
    only[columns] = 1.0
    check(model, q, k, v * only, out * only, [n], dtype)


def check_dim(model, q, k, v, out, end, dim, dtype):
    """As check() for the rows before `end` and one dim."""
    check_columns(model, q[:end], k[:end], torch.nan_to_num(v[:end], 0, 0, 0), out[:end], end, dtype, [dim])


@pytest.mark.parametrize("model", MODELS)
def test_the_largest_values_of_later_tokens_do_not_leak(gpu_ctx, model):
    """bf16 holds 3e38: a weight of a later token has to be zero, not merely small.
    (The rows that do attend them pass f32 in their sums of weights, which are up
    to 2^8 before they are divided by their own sum, and are reported.)"""
    rng = np.random.default_rng(28)
    q, k, v = inputs(rng, model, 250, BF16)
    clean = attend(gpu_ctx, model, q, k, v, [250], BF16)
    v[170:] = 3.0e38
    out = torch.zeros_like(q)
    gpu_ctx.attend_packed(model, q, k, v, out, [250])
    with pytest.raises(QxError) as e:
        gpu_ctx.sync()
    assert e.value.status == _lib.ERR_NONFINITE
    assert torch.equal(out[:170], clean[:170])


@pytest.mark.parametrize("model", MODELS)
def test_a_bad_value_at_the_end_of_a_very_long_prompt(gpu_ctx, model):
    """The rows of its tile are computed again over all their tokens, within the
    time that the rest of the kernel waits for them."""
    n = 140001
    hq, hkv, d = model_shape(model)
    gen = torch.Generator(device="cuda").manual_seed(29)
    q, k, v = (torch.randn(n, h, d, device="cuda", generator=gen).bfloat16() for h in (hq, hkv, hkv))
    clean = attend(gpu_ctx, model, q, k, v, [n], BF16)
    v[n - 1] = float("nan")
    out = torch.zeros_like(q)
    gpu_ctx.attend_packed(model, q, k, v, out, [n])
    with pytest.raises(QxError) as e:
        gpu_ctx.sync()
    assert e.value.status == _lib.ERR_NONFINITE
    assert torch.isnan(out[n - 1]).all() and torch.isfinite(out[:n - 1]).all()
    # of a mean of n values of size 1: half a step, weights rounded or not
    tol = 2.0 ** -8 * clean[n - 200:n - 1].double().abs() + (2.0 ** -8 + n * 2.0 ** -23) * 1.0
    assert ((out[n - 200:n - 1].double() - clean[n - 200:n - 1].double()).abs() <= tol).all()
    assert torch.equal(out[:n - 200], clean[:n - 200])


@pytest.mark.parametrize("model", MODELS)
def test_values_that_are_all_bad(gpu_ctx, model):
    rng = np.random.default_rng(21)
    q, k, v = inputs(rng, model, 3000, BF16)
    v[:] = float("nan")
    out = torch.zeros_like(q)
    gpu_ctx.attend_packed(model, q, k, v, out, [3000])
    with pytest.raises(QxError) as e:
        gpu_ctx.sync()
    assert e.value.status == _lib.ERR_NONFINITE and torch.isnan(out).all()


@pytest.mark.parametrize("model", MODELS)
@pytest.mark.parametrize("scale", [0.0, 30.0])
def test_flat_and_peaked_scores(gpu_ctx, model, scale):
    rng = np.random.default_rng(5)
    q, k, v = inputs(rng, model, 300, F16)
    q = q * scale
    check(model, q, k, v, attend(gpu_ctx, model, q, k, v, [300], F16), [300], F16)


@pytest.mark.parametrize("model", MODELS)
def test_rising_scores(gpu_ctx, model):
    """Each key scores higher than all before it: the running maximum moves in every tile."""
    rng = np.random.default_rng(6)
    q, k, v = inputs(rng, model, 700, F16)
    q[:] = 1.0
    k[:] = (torch.arange(700, device="cuda") / (25.0 if model == MODEL_GRANITE else 70.0))[:, None, None].half()
    check(model, q, k, v, attend(gpu_ctx, model, q, k, v, [700], F16), [700], F16)


@pytest.mark.parametrize("model,lengths", [(MODEL_GRANITE, [2500, 1100]), (MODEL_QWEN3, [3001])])
def test_long_prompts(gpu_ctx, model, lengths):
    rng = np.random.default_rng(7)
    q, k, v = inputs(rng, model, sum(lengths), BF16, fused=True)
    hq = model_shape(model)[0]
    check(model, q, k, v, attend(gpu_ctx, model, q, k, v, lengths, BF16), lengths, BF16, heads=[0, hq // 2 + 1, hq - 1])


def test_captured_and_replayed(gpu_ctx):
    rng = np.random.default_rng(8)
    lengths = [130, 1, 300]
    q, k, v = inputs(rng, MODEL_QWEN3, sum(lengths), BF16, fused=True)
    out = torch.zeros(sum(lengths), 32, 128, device="cuda", dtype=torch.bfloat16)
    old, stream = gpu_ctx.stream, torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        gpu_ctx.set_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            gpu_ctx.attend_packed(MODEL_QWEN3, q, k, v, out, lengths)
        for _ in range(2):
            q.copy_(tensor(rng, q.shape, BF16, 1.5))
            out.zero_()
            graph.replay()
            stream.synchronize()
            check(MODEL_QWEN3, q, k, v, out, lengths, BF16, heads=[0, 17])
    gpu_ctx.set_stream(old)


def test_captured_prefill_outlives_a_larger_one(gpu_ctx):
    """A captured prefill keeps its workspace when a later call needs a larger one."""
    rng = np.random.default_rng(22)
    old, stream = gpu_ctx.stream, torch.cuda.Stream()
    small = KvArena(gpu_ctx, MODEL_GRANITE, 1, 2, 40, Q4)
    q, k, v = inputs(rng, MODEL_GRANITE, 60, BF16)
    out = torch.zeros_like(q)
    go = lambda: small.prefill_packed(q, k, v, out, [40, 20], flags=_lib.DECODE_NO_ADVANCE)  # noqa: E731
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        gpu_ctx.set_stream(stream)
        go()
        stream.synchronize()
        want, rows = out.clone(), [small.read(i, 0, 0, n) for i, n in enumerate((40, 20))]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            go()
        lengths = [3000] * 40  # past any call of these tests
        large = KvArena(gpu_ctx, MODEL_GRANITE, 1, 40, 3000, Q4)
        lq, lk, lv = (torch.zeros(sum(lengths), h, 64, device="cuda", dtype=torch.bfloat16) for h in (16, 8, 8))
        large.prefill_packed(lq, lk, lv, lq.clone(), lengths)
        out.zero_()
        graph.replay()
        stream.synchronize()
    gpu_ctx.set_stream(old)
    gpu_ctx.sync()
    assert torch.equal(out, want)
    for i, n in enumerate((40, 20)):
        assert all(np.array_equal(a, b) for a, b in zip(small.read(i, 0, 0, n), rows[i]))
    small.close()
    large.close()


def test_prefill_of_more_sequences_than_a_launch_holds(gpu_ctx):
    rng = np.random.default_rng(23)
    lengths = [int(x) for x in rng.integers(0, 5, 230)]
    ids = [int(x) for x in rng.permutation(230)]
    arena = KvArena(gpu_ctx, MODEL_QWEN3, 1, 230, 5, Q4)
    q, k, v = inputs(rng, MODEL_QWEN3, sum(lengths), BF16)
    out = torch.zeros_like(q)
    arena.prefill_packed(q, k, v, out, lengths, seq_ids=ids)
    gpu_ctx.sync()
    begin = 0
    for i, n in zip(ids, lengths):
        rows = slice(begin, begin + n)
        begin += n
        assert arena.len(i) == n
        if n:
            qr, kr = (torch.from_numpy(ref.rotate64(MODEL_QWEN3, host(x[rows]), range(n), None)) for x in (q, k))
            check_rounded(MODEL_QWEN3, qr, kr, v[rows], out[rows])
            (_, _), (vc, vs) = stored(arena, i, 0, 0, n)
            want = ref.quantise(v[rows].float().cpu().numpy())
            assert np.array_equal(vc, want[0]) and np.array_equal(vs, want[1])
    arena.close()


@pytest.mark.parametrize("model", MODELS)
@pytest.mark.parametrize("page", [0, 64])
def test_prompt_then_decode(gpu_ctx, model, page):
    """Packed prompts into two layers, then three decode steps over the rows they wrote."""
    rng = np.random.default_rng([model, page, 9])
    hq, hkv, d = model_shape(model)
    qw, kw = norms(rng, model)
    lengths, ids = [37, 0, 129, 1], [2, 0, 1, 3]
    cap = max(lengths) + 3
    arena = KvArena(gpu_ctx, model, 2, 4, cap, Q4, page_size=page, pool_pages=9 if page else 0)
    for layer in range(2):
        q, k, v = inputs(rng, model, sum(lengths), BF16, fused=True)
        out = torch.zeros(sum(lengths), hq, d, device="cuda", dtype=torch.bfloat16)
        arena.prefill_packed(q, k, v, out, lengths, seq_ids=ids, layer=layer, q_norm=qw, k_norm=kw,
                             flags=_lib.DECODE_NO_ADVANCE if layer == 0 else 0)
        gpu_ctx.sync()
        begin = 0
        for i, n in zip(ids, lengths):
            rows = slice(begin, begin + n)
            begin += n
            if not n:
                continue
            qr, kr = (torch.from_numpy(ref.rotate64(model, host(x[rows]), range(n), None if w is None else host(w)))
                      for x, w in ((q, qw), (k, kw)))
            # the attention reads the rotated rows rounded to bf16
            check_rounded(model, qr, kr, v[rows], out[rows])
            (kc, ks), (vc, vs) = stored(arena, i, layer, 0, n)
            want = ref.quantise(v[rows].float().cpu().numpy())
            assert np.array_equal(vc, want[0]) and np.array_equal(vs, want[1])
            # half a code step, and the two roundings a scale and the f32 row add to it
            err = np.abs(ref.values(kc, ks) - kr.numpy()).reshape(*ks.shape, 32)
            assert (err <= 0.5 * ks.astype(np.float64)[..., None] * (1 + 2.0 ** -7) + 1e-6).all()
    assert [arena.len(i) for i in ids] == lengths
    for step in range(3):
        positions = [n + step for n in lengths]
        q, k, v = (tensor(rng, (4, 2, h, d), BF16) for h in (hq, hkv, hkv))
        out = torch.zeros(4, 2, hq, d, device="cuda")
        arena.decode(q, k, v, out, positions, seq_ids=ids, q_dtype=BF16, in_dtype=BF16, q_norm=qw, k_norm=kw)
        gpu_ctx.sync()
        check_decode(gpu_ctx, arena, q, k, v, out, positions, F32, qw, kw, ids)
    arena.close()


def check_rounded(model, q, k, v, out):
    """`out` of a prefill against 64 bits: its rotated queries and keys are
    rounded to bf16 (one step of 2^-8 each), which moves a logit by at most
    that share of |q|.|k|."""
    hq, hkv, d = model_shape(model)
    v, out, n = v.double().cpu(), out.double().cpu(), q.shape[0]
    later = torch.arange(n) > torch.arange(n)[:, None]
    for h in range(hq):
        kd, vd = k[:, h * hkv // hq], v[:, h * hkv // hq]
        p = torch.softmax((q[:, h] @ kd.T * ref.SCALE[model]).masked_fill(later, -torch.inf), -1)
        want, mean = p @ vd, p @ vd.abs()
        size = (q[:, h].abs() @ kd.abs().T).masked_fill(later, 0).amax(-1, keepdim=True) * ref.SCALE[model]
        rel = torch.expm1(2 * size * (2 * 2.0 ** -8 + (d + 16) * 2.0 ** -24)) + 2.0 ** -8 + 2.0 ** -13 + n * 2.0 ** -24
        assert float(((out[:, h] - want).abs() / (2.0 ** -8 * want.abs() + rel * mean + 1e-30)).max()) <= 1


def test_refusals(gpu_ctx):
    bad, unsupported = _lib.ERR_INVALID_ARG, _lib.ERR_UNSUPPORTED
    q, k = (torch.zeros(64, h, 64, device="cuda", dtype=torch.bfloat16) for h in (16, 8))

    def refused(status, call):
        launches = gpu_ctx.launch_count
        with pytest.raises(QxError) as e:
            call()
        assert e.value.status == status and gpu_ctx.launch_count == launches and str(e.value)
    go = lambda *a, **kw: gpu_ctx.attend_packed(kw.pop("model", MODEL_GRANITE), *a, **kw)  # noqa: E731
    refused(bad, lambda: go(q, k, k, q, []))
    refused(bad, lambda: go(q, k, k, q, [3, -1]))
    refused(bad, lambda: go(q, k, k, q, [2 ** 24, 1]))
    refused(bad, lambda: go(q.data_ptr(), k.data_ptr(), k.data_ptr(), q.data_ptr(), [2 ** 18 + 1]))
    refused(bad, lambda: go(q.data_ptr(), k.data_ptr(), k.data_ptr(), q.data_ptr(), [2 ** 18] * 64 + [1]))
    refused(bad, lambda: go(q, k, None, q, [3]))
    refused(bad, lambda: go(q, q, k, q, [3]))
    refused(bad, lambda: go(q.transpose(0, 1), k, k, q, [3]))
    refused(unsupported, lambda: go(q, k, k, q, [3], dtype=F32))
    refused(unsupported, lambda: go(q, k, k, q, [3], dtype=Q4))
    flat = torch.zeros(64 * 1024 + 8, device="cuda", dtype=torch.bfloat16)
    refused(bad, lambda: go(flat[1:1 + 64 * 1024].view(64, 16, 64), k, k, q, [3]))
    refused(bad, lambda: go(q, k, k, flat[1:1 + 64 * 1024].view(64, 16, 64), [3]))
    odd = torch.as_strided(flat, (50, 16, 64), (1028, 64, 1))
    refused(bad, lambda: go(odd, k, k, q, [3]))
    refused(bad, lambda: go(q, k[:2], k, q, [3]))
    refused(bad, lambda: go(q, k, k, q[:2], [3]))
    arena = KvArena(gpu_ctx, MODEL_GRANITE, 1, 2, 16, Q4)
    pre = lambda lengths, a=arena, **kw: a.prefill_packed(q, k, k, q.clone(), lengths, **kw)  # noqa: E731
    refused(_lib.ERR_POSITION, lambda: pre([17]))
    refused(bad, lambda: pre([1, 1], seq_ids=[0, 0]))
    refused(bad, lambda: pre([1, 1, 1]))
    refused(bad, lambda: pre([1], layer=1))
    refused(unsupported, lambda: pre([1], dtype=F32))
    refused(bad, lambda: arena.prefill_packed(q, k, k[:3], q.clone(), [2, 2]))
    refused(bad, lambda: arena.prefill_packed(q, k, k, q[:3].clone(), [2, 2]))
    plain = KvArena(gpu_ctx, MODEL_GRANITE, 1, 2, 16, BF16)
    refused(unsupported, lambda: pre([1], plain))
    pre([3, 2])
    refused(_lib.ERR_POSITION, lambda: pre([3, 2]))
    gpu_ctx.sync()
    arena.close()
    plain.close()


@pytest.mark.parametrize("model", MODELS)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_a_bad_key_reaches_every_row_that_attends_it(gpu_ctx, model, dtype):
    """Wherever in a tile it lies: the rows from it on are not finite and reported,
    the rows before it as without it. An infinite element makes a score infinite: of
    +inf nothing can be made, -inf is a weight of zero."""
    rng = np.random.default_rng([model, dtype, 32])
    lengths = [40, 300, 30]
    q, k, v = inputs(rng, model, sum(lengths), dtype)
    clean = attend(gpu_ctx, model, q, k, v, lengths, dtype)
    end = 340
    hq, hkv, _ = model_shape(model)
    for at in [40 + o for o in range(32)] + [40 + 128 + o for o in range(32)] + [339]:
        for bad in (float("nan"), float("inf")):
            keep = k[at].clone()
            if bad != bad:
                k[at] = bad
                hit = torch.ones(end - at, hq, dtype=torch.bool, device="cuda")
            else:
                k[at, :, 3] = bad
                hit = q[at:end, :, 3] > 0
            out = torch.zeros_like(clean)
            gpu_ctx.attend_packed(model, q, k, v, out, lengths, dtype=dtype)
            if hit.any():
                with pytest.raises(QxError) as e:
                    gpu_ctx.sync()
                assert e.value.status == _lib.ERR_NONFINITE
            else:
                gpu_ctx.sync()
            k[at] = keep
            finite = torch.isfinite(out[at:end])
            assert not finite[hit].any(), (at, bad)
            if bad == bad:  # its weight is 0: rows of more than one token are still means of the others
                assert finite[1:][~hit[1:]].all(), (at, bad)
            assert torch.equal(out[:at], clean[:at]) and torch.equal(out[end:], clean[end:])


@pytest.mark.parametrize("model", MODELS)
def test_a_bad_query_is_its_own_rows_affair(gpu_ctx, model):
    rng = np.random.default_rng([model, 33])
    q, k, v = inputs(rng, model, 333, BF16)
    clean = attend(gpu_ctx, model, q, k, v, [333], BF16)
    hq, _, d = model_shape(model)
    for row, head, dim in ((0, 0, 0), (77, hq - 1, d - 1), (200, 3, 17), (332, 1, 5)):
        keep = q[row, head, dim].clone()
        q[row, head, dim] = float("nan")
        out = torch.zeros_like(clean)
        gpu_ctx.attend_packed(model, q, k, v, out, [333])
        with pytest.raises(QxError) as e:
            gpu_ctx.sync()
        q[row, head, dim] = keep
        assert e.value.status == _lib.ERR_NONFINITE and not torch.isfinite(out[row, head]).any()
        out[row, head] = clean[row, head]
        assert torch.equal(out, clean)


def test_a_prefill_without_tokens(gpu_ctx):
    """Only empty prompts: nothing is launched or written, the positions still have to hold."""
    arena = KvArena(gpu_ctx, MODEL_GRANITE, 1, 3, 16, Q4)
    q, k = (torch.zeros(4, h, 64, device="cuda", dtype=torch.bfloat16) for h in (16, 8))
    out = torch.full((4, 16, 64), 5.0, device="cuda", dtype=torch.bfloat16)
    launches = gpu_ctx.launch_count
    arena.prefill_packed(q, k, k, out, [0, 0], seq_ids=[2, 0])
    arena.prefill_packed(None, None, None, None, [0])
    gpu_ctx.sync()
    assert gpu_ctx.launch_count == launches and (out == 5.0).all() and [arena.len(i) for i in range(3)] == [0, 0, 0]
    arena.prefill_packed(q, k, k, out, [4])
    with pytest.raises(QxError) as e:
        arena.prefill_packed(q, k, k, out, [0])
    assert e.value.status == _lib.ERR_POSITION
    gpu_ctx.sync()
    arena.close()


def test_a_refused_prefill_allocates_nothing(gpu_ctx):
    arena = KvArena(gpu_ctx, MODEL_GRANITE, 1, 8, 16, Q4)
    q, k = (torch.zeros(8, h, 64, device="cuda", dtype=torch.bfloat16) for h in (16, 8))
    out = torch.zeros_like(q)
    gpu_ctx.sync()
    for status, lengths, kw in ((_lib.ERR_POSITION, [2 ** 18] * 8, {}), (_lib.ERR_INVALID_ARG, [2 ** 18] * 8, {"layer": 1}),
                                (_lib.ERR_INVALID_ARG, [2 ** 18] * 8, {"seq_ids": [0] * 8})):
        free = torch.cuda.mem_get_info()[0]
        with pytest.raises(QxError) as e:
            arena.prefill_packed(q, k, k, out, lengths, **kw)
        assert torch.cuda.mem_get_info()[0] == free
        assert e.value.status in (status, _lib.ERR_POSITION)
    arena.prefill_packed(q, k, k, out, [1] * 8)
    gpu_ctx.sync()
    arena.close()


def test_a_workspace_grows_to_what_is_asked_where_more_does_not_fit():
    """With less than twice the last workspace free, a slightly larger call still runs."""
    rng = np.random.default_rng(36)
    ctx = Context(0)
    lengths = [256] * 500  # 128000 tokens, 3 KB of workspace each
    arena = KvArena(ctx, MODEL_GRANITE, 1, 500, 256, Q4)
    q, k, v = inputs(rng, MODEL_GRANITE, sum(lengths), BF16)
    out = torch.zeros_like(q)
    go = lambda n: arena.prefill_packed(q, k, v, out, lengths[:n], flags=_lib.DECODE_NO_ADVANCE)  # noqa: E731
    ctx.attend_packed(MODEL_GRANITE, q, k, v, out, lengths)  # what a first launch loads
    ctx.sync()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    hog = torch.empty(torch.cuda.mem_get_info()[0] - 950_000_000, dtype=torch.uint8, device="cuda")
    try:
        go(440)
        ctx.sync()
        assert torch.cuda.mem_get_info()[0] < 2 * 440 * 256 * 2 * (1024 + 512)
        go(500)
        ctx.sync()
    finally:
        del hog
        torch.cuda.empty_cache()
    (_, _), (vc, vs) = stored(arena, 499, 0, 0, 256)
    want = ref.quantise(v[-256:].float().cpu().numpy())
    assert np.array_equal(vc, want[0]) and np.array_equal(vs, want[1])
    arena.close()
    ctx.close()


@pytest.mark.parametrize("model", MODELS)
def test_rows_computed_again_attend_every_token(gpu_ctx, model):
    """The rows that share a tile with a bad value at the end of a long prompt, against 64
    bits. Nearly all of their weight is on 16 tokens, at the ends of the prompt and around
    the borders of the stretches that the recomputation takes, each with dims of its own:
    one left out or counted twice is off by all of its output."""
    n = 140001
    hq, hkv, d = model_shape(model)
    gen = torch.Generator(device="cuda").manual_seed(38)
    q, k, v = (torch.randn(n, h, d, device="cuda", generator=gen).bfloat16() for h in (hq, hkv, hkv))
    hot = [0, 1, 31, 32, 63, 64, 4095, 4096, 65535, 65536, 70001, 131071, n - 400, n - 257, n - 160, n - 140]
    q[:, :, 0] = 8.0
    k[:, :, 0] = 0.0
    k[hot, :, 0] = 100.0 if model == MODEL_GRANITE else 18.0  # a logit of 12.5: 2.7e5 times the others' weight
    for i, t in enumerate(hot):
        v[t] = 0.0
        v[t, :, i::16] = 8.0
    v[n - 1] = float("nan")
    out = torch.zeros_like(q)
    gpu_ctx.attend_packed(model, q, k, v, out, [n])
    with pytest.raises(QxError) as e:
        gpu_ctx.sync()
    assert e.value.status == _lib.ERR_NONFINITE and torch.isnan(out[n - 1]).all()
    rows = torch.arange(n - 1 - n % 128 - 20, n - 1, device="cuda")  # the key tile of the bad value, and some before it
    later = torch.arange(n - 1, device="cuda") > rows[:, None]
    for h in (0, hq // 2 + 1, hq - 1):
        kd, vd = k[:n - 1, h * hkv // hq].double(), v[:n - 1, h * hkv // hq].double()
        qd = q[rows, h].double()
        p = torch.softmax((qd @ kd.T * ref.SCALE[model]).masked_fill(later, -torch.inf), -1)
        want, mean = p @ vd, p @ vd.abs()
        assert float(want.abs().amax(1).min()) > 0.3  # a token's share
        size = (qd.abs() @ kd.abs().T).masked_fill(later, 0).amax(-1, keepdim=True) * ref.SCALE[model]
        rel = 2 * size * (d + 2) * 2.0 ** -24 + ref.HALF_STEP[BF16] + 2.0 ** -13 + n * 2.0 ** -24
        assert float(((out[rows, h].double() - want).abs() / (ref.HALF_STEP[BF16] * want.abs() + rel * mean)).max()) <= 1


@pytest.mark.parametrize("model", MODELS)
def test_a_bad_value_at_the_end_of_the_longest_prompt(gpu_ctx, model):
    """2^18 tokens, the most a prompt may have: no wait for the recomputed rows runs out
    (which would be another status), and the rows before its tile are as without it."""
    n = 2 ** 18
    hq, hkv, d = model_shape(model)
    gen = torch.Generator(device="cuda").manual_seed(40)
    q, k, v = (torch.randn(n, h, d, device="cuda", generator=gen).bfloat16() for h in (hq, hkv, hkv))
    clean = attend(gpu_ctx, model, q, k, v, [n], BF16)
    v[n - 1] = float("nan")
    out = torch.zeros_like(q)
    gpu_ctx.attend_packed(model, q, k, v, out, [n])
    with pytest.raises(QxError) as e:
        gpu_ctx.sync()
    assert e.value.status == _lib.ERR_NONFINITE
    assert torch.isnan(out[n - 1]).all() and torch.isfinite(out[:n - 1]).all()
    assert torch.equal(out[:n - 128], clean[:n - 128])
