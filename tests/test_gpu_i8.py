"""The 8-bit unembedding against plain 64-bit arithmetic: the norm with its 8-bit output,
the prepared weights, the product, and the chain into the sampler."""
import ctypes as C

import numpy as np
import pytest

import i8_beam_ref as ref
from vindexllm_b200 import abi, synth

pytestmark = pytest.mark.gpu

DT = {"f32": "float32", "bf16": "bfloat16", "f16": "float16"}


def _t(a, dtype=None):
    import torch
    t = torch.as_tensor(np.ascontiguousarray(a), device="cuda")
    return t if dtype is None else t.to(getattr(torch, DT[dtype]))


def _hidden(rows, dim, seed, dtype):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, dim)) * (1.0 + 20.0 * (rng.random(dim) < 0.01))
    return _t(x.astype(np.float32), dtype)


def _check_norm(q, scale, h, weight, eps):
    """q is the exact rounding; the scale is a 64-bit value rounded once to fp32 (2^-24
    relative, and below fp32's normal range half a subnormal step, 2^-150)."""
    wq, ws = ref.norm_i8(h.double().cpu().numpy(), weight.double().cpu().numpy(), eps)
    assert np.array_equal(q.cpu().numpy(), wq)
    got = scale.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(ws))
    ok = ~np.isnan(ws)
    assert (np.abs(got[ok] - ws[ok]) <= np.abs(ws[ok]) * 2.0 ** -24 * 1.001 + 2.0 ** -150).all()


@pytest.mark.parametrize("dim", [1, 7, 16, 33, 256, 1001, 1024, 2560, 3840, 8192, 8200, 32768])
@pytest.mark.parametrize("dtype", list(DT))
def test_norm(gpu_ctx, dim, dtype):
    import torch
    for rows, wtype, residual in ((1, "f32", True), (5, dtype, False), (3, "bf16", True)):
        x = _hidden(rows, dim, dim + rows, dtype)
        r = _hidden(rows, dim, dim + rows + 1, dtype) if residual else None
        w = _t(1.0 + 0.2 * np.random.default_rng(dim).standard_normal(dim).astype(np.float32), wtype)
        q, scale, h = gpu_ctx.rms_norm_i8(x, w, 1e-6, residual=r)
        want = (x.float() + r.float()).to(x.dtype) if residual else x
        if residual:
            assert torch.equal(h, want)
        else:
            assert h is None
        _check_norm(q, scale, want, w, 1e-6)


@pytest.mark.parametrize("rows", [1, 148, 149, 1000, 4099])
def test_norm_many_rows(gpu_ctx, rows):
    for dim in (72, 640, 2560):
        x, r = _hidden(rows, dim, rows, "bf16"), _hidden(rows, dim, rows + 1, "bf16")
        w = _t(np.linspace(0.5, 1.5, dim).astype(np.float32))
        q, scale, h = gpu_ctx.rms_norm_i8(x, w, 1e-5, residual=r)
        _check_norm(q, scale, (x.float() + r.float()).to(x.dtype), w, 1e-5)


def test_norm_of_fp32_products_on_a_border(gpu_ctx):
    """fp32 values times fp32 weights, 48 bits, that lie exactly on a border or next to one: 127 times
    such a product is no double. The expected steps are computed in whole numbers."""
    import torch
    from fractions import Fraction
    rng = np.random.default_rng(3)
    rows, xs, wants = 24, [], []
    v = int(rng.integers(1 << 23, 1 << 24)) | 1
    for i in range(rows):
        u = int(rng.integers(1 << 15, 1 << 16)) | 1
        # (2k + 1) u against 254 u: k + 1/2 steps; every third one is moved off its border by one unit.
        x = [(2 * k + 1) * u + (0, 1, -1)[k % 3 if i % 2 else 0] for k in range(126)] + [254 * u, -254 * u]
        x = [a * (-1) ** (i // 2 * j % 2) for j, a in enumerate(x)]
        xs.append(x)
        wants.append([round(Fraction(127 * a, 254 * u)) for a in x])  # to the even one
    w = torch.full((128,), float(v), device="cuda")
    x = torch.tensor(xs, dtype=torch.float32, device="cuda")
    want = torch.tensor(wants, dtype=torch.int8, device="cuda")
    assert (x.double().cpu() == torch.tensor(xs, dtype=torch.float64)).all()
    wide = torch.zeros(rows, 129, device="cuda")
    wide[:, 1:] = x
    for case in (x, x.repeat(20, 1), wide[:, 1:]):  # vectors, more rows than SMs, rows off the 16-byte boundary
        q, _, _ = gpu_ctx.rms_norm_i8(case, w, 1e-6)
        assert torch.equal(q, want.repeat(case.shape[0] // rows, 1))


def test_norm_about_a_row_for_each_sm(gpu_ctx):
    """Rows take more threads each while there is no more than one for every SM of this device."""
    import torch
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    for rows in (sms - 1, sms, sms + 1):
        for dim, dtype in ((640, "bf16"), (2560, "f32"), (3840, "f16")):
            x, w = _hidden(rows, dim, rows, dtype), _t(np.linspace(0.5, 1.5, dim).astype(np.float32))
            q, scale, _ = gpu_ctx.rms_norm_i8(x, w, 1e-5)
            _check_norm(q, scale, x, w, 1e-5)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("dim", [64, 72, 520, 1032, 5000, 16384, 32768])
def test_norm_many_rows_of_every_width(gpu_ctx, dtype, dim):
    """More rows than SMs, where a row takes few threads (or 1024 of them, in the widest), and rows
    that need 64 bits among ordinary ones."""
    import torch
    x = _hidden(150, dim, dim, dtype)
    x[3] = 0
    x[5, dim // 2] = float("nan")
    x[7, 1] = float("inf")
    if dtype != "f16":
        x[9] *= 1e-38
        x[11] *= 1e37
    w = _t(np.linspace(-1.5, 1.5, dim).astype(np.float32), dtype)
    q, scale, _ = gpu_ctx.rms_norm_i8(x, w, 1e-6)
    _check_norm(q, scale, x, w, 1e-6)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("dim", [40, 1001, 2560])
def test_norm_strides_in_place_and_untouched_bytes(gpu_ctx, dtype, dim):
    """Views with a row stride, a base off the 16-byte boundary, outputs in place of x and of
    the residual, and what lies behind each row's values left as it was."""
    import torch
    rows, w = 9, _t(np.linspace(-1.0, 2.0, dim).astype(np.float32))
    for off in (0, 1):
        for place in ("new", "x", "residual"):
            xb, rb = _hidden(rows, dim + 8, 1, dtype), _hidden(rows, dim + 24, 2, dtype)
            x, r = xb[:, off:off + dim], rb[:, off:off + dim]
            want = (x.float() + r.float()).to(x.dtype)
            qb = torch.full((rows, dim + 5), 77, dtype=torch.int8, device="cuda")
            target = {"new": torch.empty_like(x.contiguous()), "x": x, "residual": r}[place]
            keep = {"x": xb, "residual": rb}.get(place, xb).clone()
            q, scale, h = gpu_ctx.rms_norm_i8(x, w, 1e-6, residual=r, out_hidden=target, q=qb[:, off:off + dim])
            assert torch.equal(h, want)
            _check_norm(q, scale, want, w, 1e-6)
            assert (qb[:, :off] == 77).all() and (qb[:, off + dim:] == 77).all()
            if place != "new":
                now = xb if place == "x" else rb
                assert torch.equal(now[:, :off], keep[:, :off]) and torch.equal(now[:, off + dim:], keep[:, off + dim:])


def test_norm_hidden_without_residual_and_offset_weights(gpu_ctx):
    """The hidden state written without a residual, and weights off the 16-byte boundary."""
    import torch
    for rows in (3, 200):
        x, wb = _hidden(rows, 2048, 1, "bf16"), torch.rand(2049, device="cuda")
        for w in (wb[:2048], wb[1:]):
            out = torch.zeros_like(x)
            q, scale, h = gpu_ctx.rms_norm_i8(x, w, 1e-6, out_hidden=out)
            assert h is out and torch.equal(out, x)
            _check_norm(q, scale, x, w, 1e-6)


def test_offsets_beyond_32_bits(gpu_ctx):
    """More than 2^31 elements between the first row and the last: hidden states, 8-bit rows
    and logits."""
    import torch
    from vindexllm_b200.sampler import I8Weights
    wide = torch.empty(9, 1 << 28, dtype=torch.bfloat16, device="cuda")
    x = wide[:, 64:64 + 1040]
    x.copy_(_hidden(9, 1040, 3, "bf16"))
    w = torch.ones(1040, device="cuda")
    q8 = torch.empty(9, 1 << 28, dtype=torch.int8, device="cuda")
    q, scale, h = gpu_ctx.rms_norm_i8(x, w, 1e-6, residual=x, out_hidden=x, q=q8[:, :1040])
    _check_norm(q, scale, x, w, 1e-6)
    n, batch = 262144, 8300
    wq = torch.randint(-127, 128, (n, 1040), dtype=torch.int8, device="cuda")
    weights = I8Weights(gpu_ctx, wq, torch.ones(n, device="cuda"))
    want = (q.double() @ wq.double().T)
    got = weights.unembed(q, torch.ones(9, device="cuda"))
    assert torch.equal(got.double(), want)  # whole numbers below 2^24
    del wide, q8
    torch.cuda.empty_cache()
    rows = torch.randint(-127, 128, (batch, 1040), dtype=torch.int8, device="cuda")
    got = weights.unembed(rows, torch.ones(batch, device="cuda"), dtype=torch.bfloat16)
    assert got.numel() > 1 << 31
    for part in (slice(0, 3), slice(8190, 8195), slice(8297, 8300)):
        assert torch.equal(got[part], (rows[part].double() @ wq.double().T).to(torch.bfloat16))
    weights.close()


def test_norm_values_on_the_edge(gpu_ctx):
    """Rows of zeros, NaN, infinities, subnormals, values whose squares overflow fp32, and values on
    rounding borders (k + 1/2 of a step), which go to the even integer."""
    import torch
    dim = 254
    rows = np.ones((9, dim), np.float32)
    rows[0] = 0.0
    rows[1, 17] = np.nan
    rows[2, 253] = np.inf
    rows[3] = 1e-42
    rows[4] = 3e38 * np.linspace(-1, 1, dim)
    rows[5] = np.arange(dim) / 2.0 - 63.5
    rows[5, 0] = 127.0
    rows[6, 0] = -np.inf
    rows[7] = -0.0
    rows[8] = 1e-30
    x, w = _t(rows), torch.ones(dim, device="cuda")
    q, scale, _ = gpu_ctx.rms_norm_i8(x, w, 1e-6)
    _check_norm(q, scale, x, w, 1e-6)
    assert (q[0] == 0).all() and scale[0] == 0 and torch.isnan(scale[[1, 2, 6]]).all() and (q[[1, 2, 6]] == 0).all()
    w2 = w.clone()
    w2[3] = np.inf
    q, scale, _ = gpu_ctx.rms_norm_i8(x, w2, 1e-6)
    assert torch.isnan(scale).all() and (q == 0).all()
    q, scale, _ = gpu_ctx.rms_norm_i8(x[:1], w, 0.0)  # 0 / 0 has no rms
    assert (q == 0).all()


@pytest.mark.parametrize("dim", [64, 254, 8200])
def test_norm_of_zeros_without_eps(gpu_ctx, dim):
    """Rows and weights of zeros have scale 0 where eps is 0 too, whatever stands beside them."""
    import torch
    x = _hidden(4, dim, 3, "f32")
    x[1] = 0.0
    w = torch.ones(dim, device="cuda")
    q, scale, _ = gpu_ctx.rms_norm_i8(x, w, 0.0)
    assert scale[1] == 0 and (q[1] == 0).all()
    rest = torch.tensor([0, 2, 3], device="cuda")
    _check_norm(q[rest], scale[rest], x[rest], w, 0.0)
    q, scale, _ = gpu_ctx.rms_norm_i8(x, torch.zeros_like(w), 0.0)
    assert (scale == 0).all() and (q == 0).all()


def _ints(rows, k, seed, room=None):
    rng = np.random.default_rng(seed)
    return rng.integers(-128, 128, size=(rows, room or k)).astype(np.int8)


def _check_product(got, q, scale, wq, ws):
    """A 32-bit integer sum to fp32 (2^-24), two products (2^-24 each): 3 * 2^-24 relative
    and the subnormal step; bf16 adds its half step, 2^-8 of the value."""
    want = ref.product_i8(q, scale, wq, ws)
    rel = 3.01 * 2.0 ** -24 + (2.0 ** -8 if got.dtype != __import__("torch").float32 else 0.0)
    assert (np.abs(got.double().cpu().numpy() - want) <= np.abs(want) * rel + 1e-37).all()


@pytest.mark.parametrize("k", [1, 15, 16, 31, 32, 100, 128, 129, 640, 1000, 1152, 2560, 4112])
@pytest.mark.parametrize("batch", [1, 2, 8, 9, 16, 17, 40, 130])
def test_product(gpu_ctx, k, batch):
    import torch
    from vindexllm_b200.sampler import I8Weights
    room = -(-k // 16) * 16
    for n, dtype in ((1, torch.float32), (127, torch.bfloat16), (1000, torch.float32), (300, torch.bfloat16)):
        wq, q = _ints(n, k, k + n), _ints(batch, k, batch + k, room)
        ws, xs = np.linspace(1e-4, 2e-3, n).astype(np.float32), np.linspace(0.01, 0.2, batch).astype(np.float32)
        w = I8Weights(gpu_ctx, _t(wq), _t(ws))
        got = w.unembed(_t(q)[:, :k], _t(xs), dtype=dtype)
        _check_product(got, q[:, :k], xs, wq, ws)
        w.close()


@pytest.mark.parametrize("batch", [64, 65, 128, 200, 256, 257, 300, 515])
def test_product_larger_batches(gpu_ctx, batch):
    import torch
    from vindexllm_b200.sampler import I8Weights
    k, n = 384, 5003
    wq, q = _ints(n, k, 1), _ints(batch, k, 2)
    ws, xs = np.linspace(1e-4, 2e-3, n).astype(np.float32), np.linspace(0.01, 0.2, batch).astype(np.float32)
    w = I8Weights(gpu_ctx, _t(wq), _t(ws))
    for dtype in (torch.float32, torch.bfloat16):
        _check_product(w.unembed(_t(q), _t(xs), dtype=dtype), q, xs, wq, ws)
    w.close()


@pytest.mark.parametrize("batch,n,k", [(200, 100, 256), (200, 129, 64), (256, 128, 48), (300, 700, 2000), (1000, 257, 130),
                                       (1, 40000, 80), (77, 40001, 100), (256, 40001, 33), (513, 20001, 160),
                                       (300, 40001, 2100), (256, 1000, 8192), (144, 1000, 8192), (500, 100, 4096),
                                       (9, 1, 32768), (33, 8000, 4100), (600, 3000, 1100)])
def test_product_shapes(gpu_ctx, batch, n, k):
    """A vocabulary of one tile with a batch of two CTAs' width, the last tile of a pair half empty,
    more tiles than CTAs, several column tiles, sums split over 2, 4 and 8 CTAs, their columns in
    groups that the CTAs share unevenly."""
    import torch
    from vindexllm_b200.sampler import I8Weights
    wq, q = _ints(n, k, 1), _ints(batch, k, 2, -(-k // 16) * 16)
    ws, xs = np.linspace(1e-4, 2e-3, n).astype(np.float32), np.linspace(0.01, 0.2, batch).astype(np.float32)
    w = I8Weights(gpu_ctx, _t(wq), _t(ws))
    for dtype in (torch.float32, torch.bfloat16):
        _check_product(w.unembed(_t(q)[:, :k], _t(xs), dtype=dtype), q[:, :k], xs, wq, ws)
    gpu_ctx.device_status()
    w.close()


def test_product_on_two_streams(gpu_ctx):
    """Two calls with the same weights at once, one of them of pairs."""
    import torch
    from vindexllm_b200.sampler import I8Weights
    n, k = 60000, 512
    w = I8Weights(gpu_ctx, torch.randn(n, k, device="cuda", generator=torch.Generator("cuda").manual_seed(1)))
    q = [_t(_ints(b, k, b)) for b in (7, 300)]
    xs = [torch.rand(b.shape[0], device="cuda") for b in q]
    want = [w.unembed(a, b) for a, b in zip(q, xs)]
    streams = [torch.cuda.Stream() for _ in q]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        got = [w.unembed(a, b, stream=s) for a, b, s in zip(q, xs, streams)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    w.close()


# Products of two CTAs on a tile (test_i8_beam_host.py checks that each is one): one column tile and
# several, 160 to 256 columns (all of tensor memory), whole and partial last chunks, an odd and an
# even number of 128-entry tiles.
PAIR_SHAPES = [(129, 20001, 2048), (160, 19968, 2100), (256, 20001, 2048), (256, 19968, 2049), (512, 20001, 2560),
               (513, 20001, 2304), (512, 10000, 4096)]


@pytest.mark.parametrize("batch,n,k", PAIR_SHAPES)
def test_product_of_pairs(gpu_ctx, batch, n, k):
    import torch
    from vindexllm_b200.sampler import I8Weights
    wq, q = _ints(n, k, 1), _ints(batch, k, 2, -(-k // 16) * 16)
    ws, xs = np.linspace(1e-4, 2e-3, n).astype(np.float32), np.linspace(0.01, 0.2, batch).astype(np.float32)
    w = I8Weights(gpu_ctx, _t(wq), _t(ws))
    for dtype in (torch.float32, torch.bfloat16):
        _check_product(w.unembed(_t(q)[:, :k], _t(xs), dtype=dtype), q[:, :k], xs, wq, ws)
    gpu_ctx.device_status()
    w.close()


def test_pairs_beside_another_stream(gpu_ctx):
    """A product of pairs and one of single CTAs on two streams at once."""
    import torch
    from vindexllm_b200.sampler import I8Weights
    _, n, k = PAIR_SHAPES[2]
    w = I8Weights(gpu_ctx, torch.randn(n, k, device="cuda", generator=torch.Generator("cuda").manual_seed(1)))
    q = [_t(_ints(b, k, b)) for b in (7, 256, 300)]
    xs = [torch.rand(b.shape[0], device="cuda") for b in q]
    want = [w.unembed(a, b) for a, b in zip(q, xs)]
    streams = [torch.cuda.Stream() for _ in q]
    torch.cuda.synchronize()
    for _ in range(8):
        got = [w.unembed(a, b, stream=s) for a, b, s in zip(q, xs, streams)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    gpu_ctx.device_status()
    w.close()

def test_product_extremes(gpu_ctx):
    """The largest sums (-128 * -128 over the largest in_dim), and scales of NaN and infinity."""
    import torch
    from vindexllm_b200.sampler import I8Weights
    k, n = abi.I8_MAX_DIM, 130
    wq, q = np.full((n, k), -128, np.int8), np.full((3, k), -128, np.int8)
    q[1] = 127
    ws, xs = np.ones(n, np.float32), np.array([1.0, 2.0, np.nan], np.float32)
    ws[5] = np.inf
    w = I8Weights(gpu_ctx, _t(wq), _t(ws))
    got = w.unembed(_t(q), _t(xs)).cpu().numpy()
    assert got[0, 0] == 128.0 * 128 * k and got[1, 0] == -127.0 * 128 * k * 2 and np.isnan(got[2]).all()
    assert got[0, 5] == np.inf and got[1, 5] == -np.inf
    w.close()


def test_product_strides_and_untouched_logits(gpu_ctx):
    """Rows of q and of the logits wider than their values, the source freed, an offset base."""
    import torch
    from vindexllm_b200.sampler import I8Weights
    k, n, batch = 200, 333, 21
    wb = _ints(n, k + 9, 3)
    src = _t(wb)[:, 3:3 + k]
    ws, xs = np.linspace(1e-4, 2e-3, n).astype(np.float32), np.linspace(0.01, 0.2, batch).astype(np.float32)
    scales = _t(ws)
    w = I8Weights(gpu_ctx, src, scales)
    src.zero_()
    scales.zero_()
    qb = _ints(batch, 320, 4)
    for dtype, off in ((torch.float32, 0), (torch.float32, 1), (torch.bfloat16, 1), (torch.bfloat16, 2)):
        lb = torch.full((batch + 3, n + 7), 5.0, dtype=dtype, device="cuda")
        out = lb[:batch, off:off + n]
        got = w.unembed(_t(qb)[:, 16:16 + k], _t(xs), logits=out)
        _check_product(got, qb[:, 16:16 + k], xs, wb[:, 3:3 + k], ws)
        assert (lb[:, :off] == 5).all() and (lb[:, off + n:] == 5).all() and (lb[batch:] == 5).all()
    w.close()


@pytest.mark.parametrize("dtype", list(DT) + ["q4_0"])
def test_prepare_quantises_rows(gpu_ctx, oracle_mod, dtype):
    """Weights of other types become 8-bit rows exactly as the norm's rounding does: read back
    through products with unit vectors."""
    import torch
    from vindexllm_b200.sampler import I8Weights
    k, n = 96, 57
    if dtype == "q4_0":
        q4 = synth.make_q4_0(n, k, seed=5, device="cuda")
        w = I8Weights.from_q4_0(gpu_ctx, q4, k, n)
        b = q4.cpu().numpy().reshape(n, k // 32, 18)
        d = b[:, :, :2].copy().view(np.float16).astype(np.float64)
        nib = np.concatenate([b[:, :, 2:] & 15, b[:, :, 2:] >> 4], axis=2).astype(np.float64) - 8
        full = (nib * d).reshape(n, k)
    else:
        src = _hidden(n, k + 3, 5, dtype)[:, :k]
        src[4] = 0
        w = I8Weights(gpu_ctx, src)
        full = src.double().cpu().numpy()
    eye = np.eye(k, dtype=np.int8)
    got = w.unembed(_t(eye), torch.ones(k, device="cuda")).double().cpu().numpy().T
    top = np.abs(full).max(1)
    scale = (top / 127.0).astype(np.float32).astype(np.float64)
    q = np.where(top[:, None] > 0, np.rint(full * 127.0 / np.where(top > 0, top, 1)[:, None]), 0)
    # a whole number times a scale, rounded once
    assert (np.abs(got - q * scale[:, None]) <= np.abs(q * scale[:, None]) * 2.0 ** -24).all()
    w.close()


@pytest.mark.parametrize("batch", [1, 6, 33])
def test_sample_chain(gpu_ctx, oracle_mod, batch):
    """Norm, product and sampler in one call: the tokens of the oracle's sampler on the logits
    that the separate calls give, and the hidden state in place."""
    import torch
    from vindexllm_b200.sampler import I8Weights
    k, n = 640, 4001
    gpu_ctx.set_tie_mode(abi.TIES_FAITHFUL)
    w = I8Weights(gpu_ctx, _hidden(n, k, 8, "bf16"))
    x, r = _hidden(batch, k, 9, "bf16"), _hidden(batch, k, 10, "bf16")
    nw = _t(np.linspace(0.5, 1.5, k).astype(np.float32))
    rng = np.random.default_rng(batch)
    u = rng.random(batch).astype(np.float32)
    hist, cnt = rng.integers(0, n, size=(batch, 16)).astype(np.int32), np.full(batch, 16, np.int32)
    q, scale, h = gpu_ctx.rms_norm_i8(x, nw, 1e-6, residual=r)
    lg = w.unembed(q, scale)
    cfg = synth.sampler_config("c1", top_k=40, repeat_window=16)
    tok = w.sample(cfg, x, nw, 1e-6, residual=r, out_hidden=r, uniforms=_t(u), history=_t(hist), history_count=_t(cnt))
    assert torch.equal(r, h)
    want = oracle_mod.sample_batch(cfg, lg.cpu().numpy(), u, hist, cnt, abi.TIES_FAITHFUL)[0]
    assert (tok.cpu().numpy() == want).all()
    w.close()


def test_graph_replay_and_side_stream(gpu_ctx):
    """The chain captured after a warm-up call and replayed on new inputs; a call on a side stream;
    a capture that would have to grow the buffers is refused and the capture goes on."""
    import torch
    from vindexllm_b200.sampler import I8Weights, SamplerContext, VdxsError
    k, n, batch = 256, 2000, 12
    ctx = SamplerContext(0)
    w = I8Weights(ctx, _hidden(n, k, 1, "f32"))
    nw = torch.ones(k, device="cuda")
    cfg = synth.sampler_config("c0", temperature=0.0)
    x = _hidden(batch, k, 2, "f32")
    tok = torch.empty(batch, dtype=torch.int32, device="cuda")
    g = torch.cuda.CUDAGraph()
    with pytest.raises(VdxsError):
        with torch.cuda.graph(g):
            try:
                w.sample(cfg, x, nw, tokens=tok)
            finally:
                tok.zero_()  # the capture is still usable
    w.sample(cfg, x, nw, tokens=tok)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        w.sample(cfg, x, nw, tokens=tok)
    for seed in (3, 4):
        x.copy_(_hidden(batch, k, seed, "f32"))
        g.replay()
        torch.cuda.synchronize()
        q, scale, _ = ctx.rms_norm_i8(x, nw)
        assert torch.equal(tok.long(), w.unembed(q, scale).argmax(1))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    q, scale, _ = ctx.rms_norm_i8(x, nw, stream=side)
    lg = w.unembed(q, scale, stream=side)
    side.synchronize()
    q2, s2, _ = ctx.rms_norm_i8(x, nw)
    assert torch.equal(q, q2) and torch.equal(scale, s2) and torch.equal(lg, w.unembed(q2, s2))
    w.close()
    ctx.close()


def test_context_made_under_capture(gpu_ctx):
    """Making a context touches no stream: a capture in global mode goes on around it, work of the
    default stream is not waited for, and its first product may itself be captured."""
    import torch
    from vindexllm_b200.sampler import I8Weights, SamplerContext
    k, n, batch = 64, 300, 3
    wq, q = _ints(n, k, 1), _ints(batch, k, 2)
    w, qt, xs = I8Weights(gpu_ctx, _t(wq), torch.ones(n, device="cuda")), _t(q), torch.ones(batch, device="cuda")
    lg = torch.zeros(batch, n, device="cuda")
    torch.cuda._sleep(1 << 29)  # a quarter of a second
    mark = torch.cuda.Event()
    mark.record()
    held = SamplerContext(0)
    assert not mark.query()
    held.close()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, capture_error_mode="global"):
        ctx = SamplerContext(0)
        rc = ctx.lib.vdxs_unembed_i8(ctx.handle, w._h, qt.data_ptr(), k, xs.data_ptr(), batch, lg.data_ptr(), abi.DTYPE_F32,
                                     n, torch.cuda.current_stream().cuda_stream)
        assert rc == abi.OK
    for _ in range(2):
        lg.zero_()
        g.replay()
        ctx.device_status()
        _check_product(lg, q, np.ones(batch), wq, np.ones(n))
    w.close()

def test_refusals(gpu_ctx):
    import torch
    from vindexllm_b200.sampler import I8Weights, VdxsError
    lib, h = gpu_ctx.lib, gpu_ctx.handle
    p = lambda t: C.c_void_p(t.data_ptr())  # noqa: E731
    x, w = torch.zeros(2, 64, device="cuda"), torch.ones(64, device="cuda")
    q, s = torch.zeros(2, 64, dtype=torch.int8, device="cuda"), torch.zeros(2, device="cuda")

    def norm(xp=p(x), xs=64, rp=None, rs=64, dt=0, wp=p(w), wd=0, rows=2, dim=64, eps=1e-6, hp=None, hs=64, qp=p(q),
             qs=64, sp=p(s)):
        return lib.vdxs_rms_norm_i8(h, xp, xs, rp, rs, dt, wp, wd, rows, dim, eps, hp, hs, qp, qs, sp, None)

    assert norm() == abi.OK
    for bad in (dict(xp=None), dict(wp=None), dict(qp=None), dict(sp=None), dict(xs=63), dict(qs=63), dict(dt=3),
                dict(wd=-1), dict(rows=0), dict(dim=0), dict(eps=-1.0), dict(eps=float("nan")), dict(rp=p(x), rs=5),
                dict(hp=p(x), hs=65), dict(xp=C.c_void_p(x.data_ptr() + 2))):
        assert norm(**bad) == abi.E_INVALID_ARG, bad
    assert norm(dim=abi.I8_MAX_DIM + 1, xs=40000, qs=40000) == abi.E_UNSUPPORTED
    out = C.c_void_p()

    def prepare(wp=p(q), fmt=abi.WEIGHTS_I8, sc=p(s), stride=64, k=64, n=2):
        return lib.vdxs_i8_prepare(h, wp, fmt, sc, stride, k, n, None, C.byref(out))

    for bad in (dict(wp=None), dict(fmt=5), dict(fmt=-1), dict(sc=None), dict(stride=63), dict(k=0), dict(n=0),
                dict(fmt=abi.WEIGHTS_Q4_0, k=40)):
        assert prepare(**bad) == abi.E_INVALID_ARG and not out.value, bad
    assert prepare(k=abi.I8_MAX_DIM + 16, stride=40000) == abi.E_UNSUPPORTED
    wt = I8Weights(gpu_ctx, q, s)
    lg = torch.zeros(2, 2, device="cuda")

    def unembed(qp=p(q), qs=64, sp=p(s), b=2, lp=p(lg), dt=0, ls=2):
        return lib.vdxs_unembed_i8(h, wt._h, qp, qs, sp, b, lp, dt, ls, None)

    assert unembed() == abi.OK
    for bad in (dict(qp=None), dict(sp=None), dict(lp=None), dict(qs=48), dict(qs=72), dict(b=0), dict(dt=2), dict(ls=1),
                dict(qp=C.c_void_p(q.data_ptr() + 1))):
        assert unembed(**bad) == abi.E_INVALID_ARG, bad
    assert unembed(b=65536) == abi.E_UNSUPPORTED
    with pytest.raises(TypeError):
        wt.unembed(q.float(), s)
    with pytest.raises(ValueError):
        wt.unembed(q[:, :32], s)
    with pytest.raises(ValueError):
        I8Weights(gpu_ctx, q)
    with pytest.raises(ValueError):
        gpu_ctx.rms_norm_i8(x.cpu(), w)
    with pytest.raises(TypeError):
        gpu_ctx.rms_norm_i8(x.double(), w)
    with pytest.raises(VdxsError):
        wt.sample(synth.sampler_config("c0"), x, w)  # no uniforms
    wt.close()
