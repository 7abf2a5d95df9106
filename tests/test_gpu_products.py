"""GPU: the grouped and 8-bit products against plain evaluations in 64 bits and against the framework's own single-model product.

Tolerances, derived before the first run.  u = 2^-24 is half a step of float32.
- float32 grouped products, quantised integers and scales: equal bits.
- 8-bit products: the int32 sum is exact; its conversion and the two scalings round once each (3 u), the bias' addition once more (u of
  |v| + |b| at most, whether or not it is contracted), leaky relu's product once (u), the output type's rounding once (half its eps).
- bf16 / fp16 products: k products added in float32 in some order, each addition off by at most one step (2 u) of the sum of |h w|;
  then as above.
- Below an output type's smallest normal number its rounding is absolute: half its smallest subnormal.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_STEP = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
SUBNORMAL = {"float32": 2.0 ** -149, "bfloat16": 2.0 ** -133, "float16": 2.0 ** -24}
DTYPES = ["float32", "bfloat16", "float16"]


def _padded(x, pad):
    import torch
    if not pad:
        return x
    wide = torch.full((x.shape[0], x.shape[1] + pad), 77, dtype=x.dtype, device=x.device)
    wide[:, :x.shape[1]] = x
    return wide[:, :x.shape[1]]


def _gen(seed):
    import torch
    return torch.Generator(device="cuda:0").manual_seed(seed)


def _act64(y, act):
    import torch
    if act == "relu":
        return torch.where(y > 0, y, torch.zeros_like(y))
    if act == "leaky_relu":
        return torch.where(y > 0, y, y * float(np.float32(0.2)))
    return y


def _expect_quantized(x):
    """Definition in float64 (numpy) of the rows of a float64 array."""
    with np.errstate(all="ignore"):
        largest = np.abs(x).max(axis=1)
        s = np.maximum((largest.astype(np.float32) / np.float32(127)).astype(np.float32), np.float32(2.0 ** -126))
        q = np.clip(np.rint(x / s.astype(np.float64)[:, None]), -127, 127)
    bad = ~np.isfinite(x).all(axis=1)
    q[bad] = 0
    s[bad] = np.nan
    return q.astype(np.int8), s


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols,pad", [(1, 1, 0), (3, 1, 2), (1, 4096, 0), (257, 32, 0), (64, 33, 3), (5, 4097, 1), (33, 1000, 8), (1000, 17, 0),
                                            (7, 8200, 0), (2, 70001, 5), (4099, 64, 0), (100, 128, 4), (130, 2048, 16), (9, 516, 0)])
def test_quantize_rows(engine, dtype, rows, cols, pad):
    import torch
    x = torch.randn(rows, cols, device="cuda:0", generator=_gen(rows + cols)) * torch.exp(3 * torch.randn(rows, 1, device="cuda:0", generator=_gen(3)))
    X = _padded(x.to(getattr(torch, dtype)), pad)
    qbuf = torch.full((rows, cols + pad), 99, dtype=torch.int8, device="cuda:0")
    sbuf = torch.empty(rows, device="cuda:0")
    q, s = engine.quantize_rows(X, out=(qbuf[:, :cols], sbuf))
    wq, wsc = _expect_quantized(X.cpu().double().numpy())
    assert np.array_equal(s.cpu().numpy().view(np.uint32), wsc.view(np.uint32))
    assert np.array_equal(q.cpu().numpy(), wq)
    assert bool((qbuf[:, cols:] == 99).all())
    q2, s2 = engine.quantize_rows(X)
    assert torch.equal(q2, q) and torch.equal(s2.view(torch.int32), s.view(torch.int32))  # (an fp16 row may hold an infinity: scale NaN)


@pytest.mark.parametrize("cols", [8, 40, 300, 5000])
def test_quantize_ties_extremes_and_non_finite_rows(engine, cols):
    import torch
    rng = np.random.default_rng(cols)
    x = np.zeros((16, cols), np.float32)
    half = rng.integers(-126, 126, cols).astype(np.float32) + 0.5
    x[0] = half; x[0, 0] = 127.0                      # scale 1: every entry a tie
    x[1] = half * 2.0 ** -100; x[1, -1] = -127 * 2.0 ** -100
    x[2] = np.nextafter(half, np.float32(np.inf)); x[2, 0] = 127.0
    x[3] = np.nextafter(half, np.float32(-np.inf)); x[3, 0] = 127.0
    x[4] = rng.standard_normal(cols); x[4, 3] = np.nan
    x[5] = rng.standard_normal(cols); x[5, -1] = np.inf
    x[6] = rng.standard_normal(cols); x[6, 0] = -np.inf
    x[7] = np.nan
    x[9] = rng.standard_normal(cols) * 1e-43            # subnormal rows: the scale stops at 2^-126
    x[10] = 3.4028235e38 * rng.uniform(-1, 1, cols)
    x[11, 2] = 1.4e-45
    x[12] = -0.0
    x[13] = 127 * 2.0 ** -126 * rng.uniform(-1, 1, cols)
    x[14] = 3.0
    x[15] = rng.standard_normal(cols) * 10.0 ** rng.uniform(-30, 30)
    q, s = engine.quantize_rows(torch.from_numpy(x).cuda())
    wq, wsc = _expect_quantized(x.astype(np.float64))
    got = s.cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(wsc)) and np.array_equal(got[~np.isnan(got)], wsc[~np.isnan(wsc)])
    assert np.array_equal(q.cpu().numpy(), wq)


def _int8_inputs(rows, cin, ctot, models, seed, pad=0, extreme=False):
    import torch
    g = _gen(seed)
    h = torch.randint(-128 if extreme else -127, 128, (rows, cin), device="cuda:0", generator=g).to(torch.int8)
    w = torch.randint(-128 if extreme else -127, 128, (models, ctot, cin), device="cuda:0", generator=g).to(torch.int8)
    if extreme:
        h.fill_(-128)
        w.fill_(-128)
    hs = torch.exp(torch.randn(rows, device="cuda:0", generator=g)) * 0.01
    ws = torch.exp(torch.randn(models, ctot, device="cuda:0", generator=g)) * 0.01
    bias = torch.randn(models, ctot, device="cuda:0", generator=g)
    return _padded(h, pad), w, hs, ws, bias


def _check_int8(got, h, w, hs, ws, bias, act, dtype):
    """Rows of one model against float64."""
    acc = h.double() @ w.double().t()
    v = acc * hs.double()[:, None] * ws.double()
    y = _act64(v + (bias.double() if bias is not None else 0), act)
    b = bias.double().abs() if bias is not None else 0
    tol = 3.01 * U * v.abs() + 2.01 * U * (v.abs() + b)
    tol = tol + HALF_STEP[dtype] * (y.abs() + tol) + SUBNORMAL[dtype]
    assert bool(((got.double() - y).abs() <= tol).all()), float(((got.double() - y).abs() - tol).max())


SIZES8 = [(1, 1, 1), (1, 64, 16), (3, 16, 5), (17, 130, 33), (64, 128, 64), (65, 127, 65), (5, 4096, 300), (200, 96, 2), (300, 48, 257),
          (1, 2048, 512), (16, 1024, 96), (130, 300, 200), (515, 512, 384), (513, 1040, 520), (40, 4099, 18)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cin,ctot", SIZES8)
def test_transform_int8(engine, rows, cin, ctot, dtype):
    import torch
    for seed, (pad, use_bias, act) in enumerate([(0, False, "linear"), (16, True, "leaky_relu"), (3, True, "relu")]):
        h, w, hs, ws, bias = _int8_inputs(rows, cin, ctot, 1, 10 * rows + seed, pad)
        buf = torch.full((rows, ctot + pad), 55.0, dtype=getattr(torch, dtype), device="cuda:0")
        y = engine.transform_int8(h, hs, w[0], ws[0], bias=bias[0] if use_bias else None, act=act, out=buf[:, :ctot])
        _check_int8(y, h, w[0], hs, ws[0], bias[0] if use_bias else None, act, dtype)
        assert bool((buf[:, ctot:] == 55.0).all())
        assert torch.equal(engine.transform_int8(h, hs, w[0], ws[0], bias=bias[0] if use_bias else None, act=act, dtype=buf.dtype), y)


# one entry per tile shape and loader of the 8- and 16-bit products, per kernel for few rows, and their neighbours (an odd row, column, depth)
@pytest.mark.parametrize("rows,cin,ctot", [(8192, 4096, 4096), (8191, 4095, 4097), (4096, 2048, 2048), (4097, 2047, 2050), (9000, 1024, 2000), (8800, 1000, 2001),
                                            (100000, 512, 512), (60001, 300, 65), (1024, 4096, 4096), (1, 4096, 4096), (16, 4095, 513), (17, 2048, 700),
                                            (64, 1024, 1024), (33, 1030, 40), (200000, 128, 16), (140001, 96, 30), (131072, 64, 5)])
def test_transform_int8_large(engine, rows, cin, ctot):
    h, w, hs, ws, bias = _int8_inputs(rows, cin, ctot, 1, rows + cin)
    _check_int8(engine.transform_int8(h, hs, w[0], ws[0], bias=bias[0], act="leaky_relu"), h, w[0], hs, ws[0], bias[0], "leaky_relu", "float32")


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("rows,cin,ctot,groups", [(8192, 2048, 4096, 8), (8191, 2047, 2049, 8), (8192, 2048, 4096, 1), (2048, 1024, 1024, 64), (24, 2048, 1024, 64),
                                                   (24, 2047, 1000, 64), (5, 777, 90, 300), (300000, 32, 32, 2000), (200000, 64, 7, 300), (150000, 48, 20, 1),
                                                   (3000, 500, 500, 257), (20000, 200, 120, 256)])
def test_grouped_half_precision_large(engine, rows, cin, ctot, groups, dtype):
    """Uneven groups (some empty); every group its own weights, or one of eight models."""
    import torch
    rng = np.random.default_rng(rows)
    cut = np.sort(rng.integers(0, rows + 1, groups - 1)) if groups > 1 else np.zeros(0, int)
    sizes = np.diff(np.concatenate([[0], cut, [rows]])).tolist()
    ptr, blocks = _groups(sizes)
    M = groups if groups <= 64 else 8
    of = [g if groups <= 64 else int(rng.integers(0, M)) for g in range(groups)]
    g, t = _gen(cin), getattr(torch, dtype)
    H = torch.randn(rows, cin, device="cuda:0", generator=g).to(t)
    W = torch.randn(M, ctot, cin, device="cuda:0", generator=g).to(t)
    y = engine.transform_grouped(H, W, ptr, model_of_group=None if groups <= 64 else torch.tensor(of, dtype=torch.int32, device="cuda:0"))
    of_row = torch.repeat_interleave(torch.tensor(of), torch.tensor(sizes)).cuda()
    for m in range(M):
        idx = torch.nonzero(of_row == m).flatten()
        if idx.numel() == 0:
            continue
        h, w = H[idx].double(), W[m].double()
        want, mag = h @ w.t(), h.abs() @ w.abs().t()
        tol = 2.01 * U * cin * mag
        tol = tol + HALF_STEP[dtype] * (want.abs() + tol) + SUBNORMAL[dtype]
        assert bool(((y[idx].double() - want).abs() <= tol).all()), m


@pytest.mark.parametrize("rows,cin,ctot,groups", [(8192, 256, 1024, 1), (8191, 257, 1023, 1), (800000, 32, 2, 4000), (140000, 16, 32, 300), (131072, 8, 17, 257), (50000, 100, 20, 250),
                                                   (16, 1024, 600, 16), (1, 4096, 33, 1), (300, 31, 65, 7)])
def test_grouped_float32_large(engine, rows, cin, ctot, groups):
    import torch
    rng = np.random.default_rng(rows)
    cut = np.sort(rng.integers(0, rows + 1, groups - 1)) if groups > 1 else np.zeros(0, int)
    sizes = np.diff(np.concatenate([[0], cut, [rows]])).tolist()
    ptr, blocks = _groups(sizes)
    of = [int(x) for x in rng.integers(0, 3, groups)]
    H = torch.randn(rows, cin, device="cuda:0", generator=_gen(cin))
    W = torch.randn(3, ctot, cin, device="cuda:0", generator=_gen(1))
    of_row = torch.repeat_interleave(torch.tensor(of), torch.tensor(sizes)).cuda()
    for precise in (False, True):
        y = engine.transform_grouped(H, W, ptr, model_of_group=torch.tensor(of, dtype=torch.int32, device="cuda:0"), precise=precise)
        for m in range(3):
            full = engine.transform(H, W[m].t().contiguous(), precise=precise)
            assert torch.equal(y[of_row == m], full[of_row == m])


def test_int8_sums_are_exact_at_the_largest_depth(engine):
    import torch
    rows, cin, ctot = 3, 131071, 5
    h, w, hs, ws, _ = _int8_inputs(rows, cin, ctot, 1, 1, extreme=True)
    y = engine.transform_int8(h, torch.ones_like(hs), w[0], torch.ones_like(ws[0]))
    assert bool((y == float(np.float32(16384 * cin))).all())
    assert bool((engine.transform_int8(h[:, :300].contiguous(), torch.ones_like(hs), w[0, :, :300].contiguous(), torch.ones_like(ws[0])) == 16384.0 * 300).all())


def test_nan_scale_spreads_over_its_row_only(engine):
    import torch
    x = torch.randn(9, 64, device="cuda:0", generator=_gen(0))
    x[4, 7] = float("inf")
    q, s = engine.quantize_rows(x)
    wq, ws = engine.quantize_rows(torch.randn(33, 64, device="cuda:0", generator=_gen(1)))
    for act in ("linear", "leaky_relu"):
        y = engine.transform_int8(q, s, wq, ws, act=act)
        assert bool(torch.isnan(y[4]).all()) and not bool(torch.isnan(y[[0, 1, 2, 3, 5, 6, 7, 8]]).any())


def _groups(sizes, front=0):
    import torch
    ptr = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32) + front
    return torch.from_numpy(ptr).cuda(), [(int(a), int(b)) for a, b in zip(ptr, ptr[1:])]


GROUPS = {
    "one": [150], "empties": [0, 3, 0, 0, 70, 1, 0, 64, 65, 0], "singles": [1] * 70, "graphs": [100 + 17 * (i % 9) for i in range(30)],
    "uneven": [700, 2, 0, 33, 16, 17, 129], "many": [(i * 7) % 3 for i in range(4200)], "none": [0, 0, 0],
}


@pytest.mark.parametrize("name", sorted(GROUPS))
@pytest.mark.parametrize("cin,ctot", [(1, 64), (32, 64), (32, 2), (33, 40), (128, 256), (5, 3), (200, 130), (64, 16)])
def test_grouped_float32_has_the_single_models_bits(engine, name, cin, ctot):
    """Against ``transform`` (ascending chain), per group; rows in front of and behind the groups stay as they were."""
    import torch
    sizes = GROUPS[name]
    front, behind, M = 5, 9, 3
    rows = front + sum(sizes) + behind
    ptr, blocks = _groups(sizes, front)
    g = _gen(cin)
    H = torch.randn(rows, cin, device="cuda:0", generator=g)
    W = torch.randn(M, ctot, cin, device="cuda:0", generator=g)
    bias = torch.randn(M, ctot, device="cuda:0", generator=g)
    of = [(i * 5) % M for i in range(len(sizes))]
    mog = torch.tensor(of, dtype=torch.int32, device="cuda:0")
    full = {p: [engine.transform(H, W[m].t().contiguous(), precise=p) for m in range(M)] for p in (False, True)}
    for precise, pad, use_bias, act in [(False, 0, False, "linear"), (True, 0, False, "linear"), (False, 3, True, "leaky_relu"), (True, 1, True, "relu"),
                                        (False, 4, False, "relu")]:
        buf = torch.full((rows, ctot + pad), 55.0, device="cuda:0")
        y = engine.transform_grouped(_padded(H, pad), W, ptr, model_of_group=mog, bias=bias if use_bias else None, act=act, precise=precise,
                                     out=buf[:, :ctot])
        want = torch.full((rows, ctot), 55.0, device="cuda:0")
        for (lo, hi), m in zip(blocks, of):
            v = full[precise][m][lo:hi]
            v = v + bias[m] if use_bias else v
            want[lo:hi] = torch.where(v > 0, v, v * 0 if act == "relu" else v * 0.2 if act == "leaky_relu" else v)
        assert torch.equal(y, want), (precise, pad, act)
        assert bool((buf[:, ctot:] == 55.0).all())


def test_grouped_constant_features(engine):
    import torch
    ptr, blocks = _groups([10, 0, 80, 3])
    W = torch.randn(4, 64, 19, device="cuda:0", generator=_gen(2))
    y = engine.transform_grouped(None, W, ptr, rows=93, h_const=float(np.float32(1 / 19)))
    for g, (lo, hi) in enumerate(blocks):
        if hi > lo:
            assert torch.equal(y[lo:hi], engine.transform(None, W[g].t().contiguous(), rows=hi - lo, h_const=float(np.float32(1 / 19))))
    p = engine.transform_grouped(None, W, ptr, rows=93, h_const=0.3, precise=True)
    assert torch.equal(p[:10], engine.transform(None, W[0].t().contiguous(), rows=10, h_const=0.3, precise=True))


@pytest.mark.parametrize("rows,cin,ctot", [(3, 64, 20), (70, 64, 70), (5, 512, 64), (300, 700, 130), (140000, 64, 16)])
def test_subnormal_inputs_count(engine, rows, cin, ctot):
    """fp16 values below 2^-14 and bf16 / float32 values below 2^-126 enter the products as they are (the sums here are exact)."""
    import torch
    ptr, _ = _groups([rows])
    for dtype, tiny in ((torch.float16, 2.0 ** -24), (torch.bfloat16, 2.0 ** -133), (torch.float32, 2.0 ** -149)):
        H = torch.full((rows, cin), tiny, dtype=dtype, device="cuda:0")
        W = torch.full((1, ctot, cin), 2.0, dtype=dtype, device="cuda:0")
        y = engine.transform_grouped(H, W, ptr)
        assert bool((y.double() == 2 * cin * tiny).all()), dtype


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("name", sorted(GROUPS))
@pytest.mark.parametrize("cin,ctot", [(1, 64), (64, 64), (96, 2), (33, 41), (512, 260), (2000, 72)])
def test_grouped_half_precision(engine, name, cin, ctot, dtype):
    import torch
    sizes = GROUPS[name]
    rows, M = sum(sizes) + 4, max(1, min(len(sizes), 6))
    ptr, blocks = _groups(sizes, 4)
    g, t = _gen(cin + 1), getattr(torch, dtype)
    H = torch.randn(rows, cin, device="cuda:0", generator=g).to(t)
    W = torch.randn(M, ctot, cin, device="cuda:0", generator=g).to(t)
    bias = torch.randn(M, ctot, device="cuda:0", generator=g)
    of = [(i * 7) % M for i in range(len(sizes))]
    mog = torch.tensor(of, dtype=torch.int32, device="cuda:0")
    for pad, use_bias, act in [(0, False, "linear"), (1, True, "leaky_relu"), (8, True, "relu")]:
        buf = torch.full((rows, ctot + pad), 55.0, dtype=t, device="cuda:0")
        y = engine.transform_grouped(_padded(H, pad), W, ptr, model_of_group=mog, bias=bias if use_bias else None, act=act, out=buf[:, :ctot])
        of_row = torch.repeat_interleave(torch.tensor(of + [0]), torch.tensor(sizes + [0])).cuda()
        for m in range(M):
            idx = torch.nonzero(of_row == m).flatten() + 4
            h, w = H[idx].double(), W[m].double()
            v, mag = h @ w.t(), h.abs() @ w.abs().t()
            b = bias[m].double() if use_bias else torch.zeros(ctot, dtype=torch.float64, device="cuda:0")
            want = _act64(v + b, act)
            tol = 2.01 * U * cin * mag + 2.01 * U * (v.abs() + b.abs())
            tol = tol + HALF_STEP[dtype] * (want.abs() + tol) + SUBNORMAL[dtype]
            assert bool(((y[idx].double() - want).abs() <= tol).all()), (m, act)
        assert bool((buf[:, ctot:] == 55.0).all()) and bool((buf[:4] == 55.0).all())


@pytest.mark.parametrize("name", sorted(GROUPS))
@pytest.mark.parametrize("cin,ctot", [(1, 3), (64, 64), (130, 66), (512, 260), (2000, 72)])
def test_grouped_int8(engine, name, cin, ctot):
    import torch
    sizes = GROUPS[name]
    rows, M = sum(sizes) + 7, max(1, min(len(sizes), 5))
    ptr, blocks = _groups(sizes, 0)
    of = [(i * 3) % M for i in range(len(sizes))]
    mog = torch.tensor(of, dtype=torch.int32, device="cuda:0")
    of_row = torch.repeat_interleave(torch.tensor(of + [0]), torch.tensor(sizes + [0])).cuda()
    for seed, (pad, use_bias, act, dtype) in enumerate([(0, False, "linear", "float32"), (16, True, "leaky_relu", "bfloat16"), (5, True, "relu", "float16")]):
        h, w, hs, ws, bias = _int8_inputs(rows, cin, ctot, M, seed, pad)
        buf = torch.full((rows, ctot + pad), 55.0, dtype=getattr(torch, dtype), device="cuda:0")
        y = engine.transform_grouped_int8(h, hs, w, ws, ptr, model_of_group=mog, bias=bias if use_bias else None, act=act, out=buf[:, :ctot])
        for m in range(M):
            idx = torch.nonzero(of_row == m).flatten()
            _check_int8(y[idx], h[idx], w[m], hs[idx], ws[m], bias[m] if use_bias else None, act, dtype)
        assert bool((buf[:, ctot:] == 55.0).all()) and bool((buf[sum(sizes):] == 55.0).all())


def test_non_finite_values_stay_in_their_row_and_column(engine):
    """An infinity or NaN of H reaches its own row, one of W its own column - no padding, tail or neighbour."""
    import torch
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        for rows, cin, ctot in [(70, 36, 50), (3, 100, 20), (300, 129, 140), (9, 64, 64)]:
            H = torch.randn(rows, cin, device="cuda:0", generator=_gen(1)).to(dtype)
            W = torch.randn(1, ctot, cin, device="cuda:0", generator=_gen(2)).to(dtype)
            H[1, cin - 1], H[2, 0] = float("nan"), float("inf")
            W[0, 3, cin - 1], W[0, ctot - 1, 1] = float("inf"), float("nan")
            ptr, _ = _groups([rows])
            bad = ~torch.isfinite(engine.transform_grouped(H, W, ptr).float())
            want = torch.zeros_like(bad)
            want[1], want[2], want[:, 3], want[:, ctot - 1] = True, True, True, True
            assert torch.equal(bad, want), (dtype, rows)


@pytest.mark.parametrize("rows,cin,ctot", [(9, 64, 33), (40, 1024, 64), (300, 200, 130), (140000, 64, 16)])
def test_nan_passes_every_activation(engine, rows, cin, ctot):
    import torch
    x = torch.randn(rows, cin, device="cuda:0", generator=_gen(3))
    x[4, 5] = float("nan")
    ptr, _ = _groups([rows])
    W = torch.randn(1, ctot, cin, device="cuda:0", generator=_gen(4))
    q, s = engine.quantize_rows(x)
    wq, ws = engine.quantize_rows(W[0])
    want = torch.zeros(rows, ctot, dtype=torch.bool, device="cuda:0")
    want[4] = True
    for act in ("linear", "leaky_relu", "relu"):
        for y in (engine.transform_int8(q, s, wq, ws, act=act), engine.transform_grouped(x, W, ptr, act=act), engine.transform_grouped(x, W, ptr, act=act, precise=True),
                  engine.transform_grouped(x.half(), W.half(), ptr, act=act)):
            assert torch.equal(torch.isnan(y), want), act


def test_bad_groups_are_reported_and_leave_their_rows(engine):
    import torch
    from distgcn_amd._lib import DgcnError
    H, W = torch.randn(40, 16, device="cuda:0", generator=_gen(1)), torch.randn(2, 8, 16, device="cuda:0", generator=_gen(2))
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda:0")
    good = engine.transform_grouped(H, W, i32([0, 10, 20, 40]), model_of_group=i32([0, 1, 0]))
    for bad_id in (-1, 2, 2 ** 31 - 1):
        out, status = torch.full((40, 8), 55.0, device="cuda:0"), i32([0])
        engine.transform_grouped(H, W, i32([0, 10, 20, 40]), model_of_group=i32([0, bad_id, 0]), out=out, status=status)
        assert int(status) == 32 and bool((out[10:20] == 55.0).all())
        assert torch.equal(out[:10], good[:10]) and torch.equal(out[20:], good[20:])
        with pytest.raises(DgcnError, match="model id"):
            engine.transform_grouped(H, W, i32([0, 10, 20, 40]), model_of_group=i32([0, bad_id, 0]))
    hq, hs = engine.quantize_rows(H)
    wq, ws = engine.quantize_rows(W.reshape(16, 16))
    for ptr in ([0, 30, 20, 40], [0, 10, 20, 41], [-1, 10, 20, 40], [0, 10, 2 ** 31 - 1, 40], [0, -(2 ** 31), 20, 40]):
        with pytest.raises(DgcnError, match="row range"):
            engine.transform_grouped(H, W, i32(ptr), model_of_group=i32([0, 1, 0]))
        with pytest.raises(DgcnError, match="row range"):
            engine.transform_grouped_int8(hq, hs, wq.reshape(2, 8, 16), ws.reshape(2, 8), i32(ptr), model_of_group=i32([0, 1, 0]))


def test_offsets_beyond_32_bits(engine):
    """Three rows 1.5e9 elements apart: the last ones start behind 2^31 bytes."""
    import torch
    ld = 1_500_000_000
    buf = torch.empty(2 * ld + 128, dtype=torch.int8, device="cuda:0")
    h, w, hs, ws, _ = _int8_inputs(3, 64, 20, 1, 4)
    H = torch.as_strided(buf, (3, 64), (ld, 1))
    H.copy_(h)
    assert torch.equal(engine.transform_int8(H, hs, w[0], ws[0]), engine.transform_int8(h, hs, w[0], ws[0]))
    Y = torch.as_strided(buf.view(torch.int16)[:ld + 64].view(torch.bfloat16), (3, 20), (ld // 2, 1))
    engine.transform_int8(h, hs, w[0], ws[0], out=Y)
    assert torch.equal(Y, engine.transform_int8(h, hs, w[0], ws[0], dtype=torch.bfloat16))
    x = torch.randn(3, 64, device="cuda:0", generator=_gen(1)).half()
    X = torch.as_strided(buf.view(torch.float16), (3, 64), (ld // 2, 1))
    X.copy_(x)
    q, s = engine.quantize_rows(X)
    q2, s2 = engine.quantize_rows(x)
    assert torch.equal(q, q2) and torch.equal(s, s2)


# ---- together: a layer of a mixed batch, captured, on other streams; whole models ------------------------------------------------------

def _layer(engine, s):
    q, hs = engine.quantize_rows(s["H"])
    return [q, hs, engine.transform_grouped_int8(q, hs, s["wq"], s["ws"], s["ptr"], model_of_group=s["mog"], bias=s["bias"], act="leaky_relu", status=s["status"]),
            engine.transform_grouped(s["H"], s["W"], s["ptr"], model_of_group=s["mog"], status=s["status"]),
            engine.transform_grouped(s["H"].bfloat16(), s["W"].bfloat16(), s["ptr"], model_of_group=s["mog"], status=s["status"]),
            engine.transform_int8(q, hs, s["wq"][0], s["ws"][0])]


def _layer_state(engine, seed, sizes, cin=96, ctot=130):
    import torch
    g = _gen(seed)
    ptr, _ = _groups(sizes)
    W = torch.randn(3, ctot, cin, device="cuda:0", generator=g)
    wq, ws = engine.quantize_rows(W.reshape(-1, cin))
    return {"H": torch.randn(sum(sizes), cin, device="cuda:0", generator=g), "W": W, "wq": wq.reshape(W.shape), "ws": ws.reshape(3, ctot), "ptr": ptr,
            "mog": torch.tensor([i % 3 for i in range(len(sizes))], dtype=torch.int32, device="cuda:0"),
            "bias": torch.randn(3, ctot, device="cuda:0", generator=g), "status": torch.zeros(1, dtype=torch.int32, device="cuda:0")}


@pytest.mark.parametrize("sizes", [[100, 0, 300, 7], [1, 2, 1, 0, 3]])
def test_captured_layer_follows_its_inputs(engine, sizes):
    import torch
    s = _layer_state(engine, 1, sizes)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _layer(engine, s)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = _layer(engine, s)
    for seed in range(4):
        s["H"].copy_(torch.randn(s["H"].shape, device="cuda:0", generator=_gen(50 + seed)))
        if seed == 2:  # other groups: the table is read when the graph runs
            s["ptr"].copy_(torch.tensor([0] + [s["H"].shape[0] * (i + 1) // len(sizes) for i in range(len(sizes))], dtype=torch.int32))
        graph.replay()
        got = [o.clone() for o in outs]
        torch.cuda.synchronize()
        for a, b in zip(got, _layer(engine, s)):
            assert torch.equal(a, b)
        assert int(s["status"]) == 0


def test_two_streams_at_once(engine):
    import torch
    states = [_layer_state(engine, 2, [200, 90, 0, 411]), _layer_state(engine, 3, [1, 1, 5, 0, 2, 700])]
    want = [_layer(engine, s) for s in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    runs = []
    for _ in range(10):
        for st, s in zip(streams, states):
            with torch.cuda.stream(st):
                runs.append(_layer(engine, s))
    torch.cuda.synchronize()
    for i, outs in enumerate(runs):
        for a, b in zip(outs, want[i % 2]):
            assert torch.equal(a, b)


def _mixed_batch(engine, B=24, seed=3):
    import torch
    import scipy.sparse as sp
    from distgcn_amd.batch import HostBatch
    rng = np.random.default_rng(seed)
    adjs, wts = [], []
    for i in range(B):
        n = [0, 1, 2, 5, 60, 100, 150, 200][i % 8]
        a = np.triu(rng.random((n, n)) < 0.1, 1)
        adjs.append(sp.csr_matrix((a + a.T).astype(float)))
        wts.append(rng.random(n))
    hb = HostBatch.from_scipy(adjs, wts)
    of = rng.integers(0, 3, B).astype(np.int32)
    return hb, engine.upload(hb), of, torch.from_numpy(of).cuda()


@pytest.mark.parametrize("hidden,layers,feat", [(32, 20, 1), (32, 1, 1), (16, 3, 4), (64, 5, 1), (19, 4, 1)])
def test_bank_equals_every_graph_with_its_own_model(engine, hidden, layers, feat):
    import torch
    from distgcn_amd import datagen
    from distgcn_amd.engine import DeviceModel
    hb, db, of, mog = _mixed_batch(engine)
    models = [datagen.random_model(layers, hidden, feature_size=feat, seed=s) for s in (1, 2, 3)]
    bank = engine.model_bank(models)
    X = None if feat == 1 else torch.randn(hb.num_nodes, feat, device="cuda:0", generator=_gen(9))
    scores = engine.forward_bank(db, bank, mog, X=X)
    sol = engine.solve_bank(db, bank, mog, X=X)
    engine.check_status(sol["status"])
    assert torch.equal(sol["scores"], scores)
    for m in range(3):
        ref = engine.solve(db, DeviceModel(models[m], "cuda:0"), X=X)
        for g, (lo, hi) in enumerate(hb.graph_slices()):
            if of[g] == m:
                assert torch.equal(scores[lo:hi], ref["scores"][lo:hi]), (g, m)
                assert torch.equal(sol["state"][lo:hi], ref["state"][lo:hi])
                assert float(sol["totals"][g]) == float(ref["totals"][g])


def test_bank_with_biases_is_close(engine):
    """A bank adds its biases in front of the neighbours' sum, a single model behind it: two float32 orders of the same few terms,
    three layers deep.  Against float64 of the formula both stay within the library's 1e-5 bar for shallow stacks."""
    import torch
    from distgcn_amd import datagen
    from distgcn_amd.engine import DeviceModel
    hb, db, of, mog = _mixed_batch(engine)
    models = [datagen.random_model(3, 16, bias=True, seed=s) for s in (4, 5, 6)]
    scores = engine.forward_bank(db, engine.model_bank(models), mog)
    for m in range(3):
        ref = engine.forward(db, DeviceModel(models[m], "cuda:0"))
        for g, (lo, hi) in enumerate(hb.graph_slices()):
            if of[g] == m and hi > lo:
                assert float((scores[lo:hi] - ref[lo:hi]).abs().max()) <= 1e-5


@pytest.mark.parametrize("hidden", [32, 48])
def test_int8_bank_is_the_written_formula(engine, hidden):
    """Three layers: float32 first layer, quantised hidden layer, float32 last layer, every step restated on the host (the integer
    sums in int64, the scalings in float32, the aggregations by the twin): equal bits."""
    import torch
    from distgcn_amd import datagen
    from oracle import ctwin
    hb, db, of, mog = _mixed_batch(engine)
    models = [datagen.random_model(3, hidden, seed=s) for s in (7, 8, 9)]
    scores = engine.forward_bank(db, engine.model_bank(models, precision="int8"), mog).cpu().numpy()
    lrp, lc, lv, _ = ctwin.supports(hb.graph_ptr, hb.row_ptr, hb.col_idx)
    first = engine.forward_bank(db, engine.model_bank([m[:1] for m in models]), mog).cpu().numpy()
    q, s = _expect_quantized(first.astype(np.float64))
    of_row = np.repeat(of, np.diff(hb.graph_ptr))
    Z = np.zeros((hb.num_nodes, 2 * hidden), np.float32)
    for m in range(3):
        w = np.concatenate(models[m][1]["weights"], axis=1).T
        wq, wsc = _expect_quantized(w.astype(np.float64))
        acc = q.astype(np.int64) @ wq.T.astype(np.int64)
        z = (acc.astype(np.float32) * s[:, None]) * wsc
        Z[of_row == m] = z[of_row == m]
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
    lap = engine.supports(db)
    H = engine.spmm(lap, dev(Z[:, hidden:]), hidden, graph_ptr=db.graph_ptr, num_graphs=hb.num_graphs, max_nodes=hb.max_nodes, Y0=dev(Z), ldy0=2 * hidden,
                    act="leaky_relu")
    want = np.zeros((hb.num_nodes, 1), np.float32)
    for m in range(3):
        z = engine.transform(H, dev(np.concatenate(models[m][2]["weights"], axis=1)))
        y = engine.spmm(lap, z[:, 1:].contiguous(), 1, graph_ptr=db.graph_ptr, num_graphs=hb.num_graphs, max_nodes=hb.max_nodes, Y0=z, ldy0=2).cpu().numpy()
        want[of_row == m] = y[of_row == m]
    assert np.array_equal(scores, want)


@pytest.mark.parametrize("precision", ["float32", "int8"])
def test_captured_bank_follows_its_inputs(engine, precision):
    """A whole forward pass in a graph: replays with other features and other models per graph, eager work between them."""
    import torch
    from distgcn_amd import datagen
    from distgcn_amd._lib import DgcnError
    hb, db, of, mog = _mixed_batch(engine)
    bank = engine.model_bank([datagen.random_model(4, 24, feature_size=4, seed=i) for i in range(3)], precision=precision)
    X = torch.randn(hb.num_nodes, 4, device="cuda:0", generator=_gen(1))
    status = torch.zeros(1, dtype=torch.int32, device="cuda:0")
    with pytest.raises(DgcnError, match="before the capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.zeros(1, device="cuda:0")
            engine.forward_bank(db, bank, mog, X=X, status=status)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        engine.forward_bank(db, bank, mog, X=X, status=status)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = engine.forward_bank(db, bank, mog, X=X, status=status)
    for seed in range(4):
        X.copy_(torch.randn(X.shape, device="cuda:0", generator=_gen(60 + seed)))
        mog.copy_((mog + 1) % 3)
        graph.replay()
        got = out.clone()
        torch.cuda.synchronize()
        assert torch.equal(got, engine.forward_bank(db, bank, mog, X=X, status=status))
        assert int(status) == 0


def test_bank_reports_a_wrong_model_id(engine):
    import torch
    from distgcn_amd import datagen
    from distgcn_amd._lib import DgcnError
    hb, db, of, mog = _mixed_batch(engine)
    bank = engine.model_bank([datagen.random_model(2, 8, seed=1)])
    with pytest.raises(DgcnError, match="model id"):
        engine.forward_bank(db, bank, mog)
    with pytest.raises(ValueError):
        engine.forward_bank(db, bank, mog[:-1].contiguous())
    bank = engine.model_bank([datagen.random_model(2, 8, seed=i) for i in range(3)])
    with pytest.raises(ValueError, match="engine on"):
        engine.transform_grouped(torch.zeros(3, 1), bank.layers[0]["weights"], db.graph_ptr)
