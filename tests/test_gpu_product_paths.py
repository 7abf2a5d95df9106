"""GPU: every kernel that the dense products choose from - each tile shape with both of its loaders, the kernels for few and for many rows -
against 64 bits, with every output type, biases, activations and padded matrices.  (tests/test_product_paths.py holds that the calls
here reach all of them.)  Tolerances as in test_gpu_products.py."""
import numpy as np
import pytest

from test_gpu_products import HALF_STEP, SUBNORMAL, U, _act64, _check_int8, _gen, _groups, _int8_inputs, _padded

pytestmark = pytest.mark.gpu

# (rows, cin, ctot, groups; 0: the product of one model without a table)
INT8 = [(600, 130, 300, 0), (600, 128, 300, 0), (2048, 512, 2050, 64), (1024, 2048, 2048, 0), (513, 511, 4096, 8), (2000, 1024, 1024, 30), (1024, 4096, 4096, 0), (16384, 2001, 2050, 64),
        (4096, 2047, 2047, 0), (4096, 2048, 2048, 0), (12000, 2048, 257, 64), (4097, 2047, 2050, 64), (4096, 2048, 2050, 8), (8192, 2048, 4096, 0), (16384, 512, 700, 8),
        (17, 2048, 700, 0), (40, 1030, 70, 5), (3, 2050, 100, 0), (9, 1030, 50, 0), (140000, 64, 13, 3), (140000, 96, 30, 200)]
HALF = [(600, 65, 300, 5), (600, 64, 300, 5), (1000, 1023, 700, 64), (2048, 1024, 1030, 64), (2048, 255, 2050, 8), (4096, 1023, 2047, 1), (4096, 1024, 2048, 1),
        (12000, 1024, 257, 64), (4096, 1023, 2050, 64), (8192, 1024, 1025, 8), (16384, 64, 700, 8), (8192, 2048, 4096, 1), (40, 515, 70, 5), (140000, 32, 13, 3),
        (140000, 48, 30, 200)]
F32 = [(5000, 40, 13, 6), (5000, 41, 13, 6), (5000, 40, 30, 6), (5000, 41, 30, 6), (5000, 32, 60, 6), (5000, 31, 60, 6), (5000, 48, 100, 6), (5000, 49, 100, 6),
       (8192, 256, 1024, 1), (8191, 257, 1023, 1), (140000, 32, 13, 7), (140000, 16, 30, 7)]
# columns behind a row of the strided matrices: rows of H stay at multiples of 16 bytes with the first, and never with the second
PADS = [(0, "linear"), (16, "leaky_relu"), (3, "relu")]


def _table(rows, groups):
    """Uneven groups, some empty -> (pointers, [(first, last)], model of each: at most 8 models)."""
    import torch
    rng = np.random.default_rng(rows + groups)
    cut = np.sort(rng.integers(0, rows + 1, groups - 1)) if groups > 1 else np.zeros(0, int)
    ptr, blocks = _groups(np.diff(np.concatenate([[0], cut, [rows]])).tolist())
    of = rng.integers(0, min(groups, 8), groups).astype(np.int32)
    return ptr, blocks, torch.from_numpy(of).cuda(), of.tolist()


def _check_int8_with_overflow(got, h, w, hs, ws, bias, act, dtype):
    """The scales here reach beyond fp16: its largest number is 65 504, the next would be 65 536, and rounding to nearest turns |x| >= 65 520
    into an infinity.  One is right where the value may be that large before its last rounding (its float32 error: at most 5.02 u of
    |v| + |b|, with |v| <= 5 (|y| + |b|) - leaky relu leaves at least a fifth - and u = 2^-24); everything else as without."""
    import torch
    if dtype == "float16":
        b = bias.double() if bias is not None else torch.zeros(w.shape[0], dtype=torch.float64, device=w.device)
        y = _act64((h.double() @ w.double().t()) * hs.double()[:, None] * ws.double() + b, act)
        large = y.abs() + 5.02 * U * (5 * y.abs() + 6 * b.abs()) >= 65520
        got = torch.where(torch.isinf(got) & large & (got.sign() == y.sign()), y, got.double())
    _check_int8(got, h, w, hs, ws, bias, act, dtype)


@pytest.mark.parametrize("rows,cin,ctot,groups", INT8)
def test_int8(engine, rows, cin, ctot, groups):
    import torch
    M = max(1, min(groups, 8))
    ptr, blocks, mog, of = _table(rows, max(groups, 1))
    for (pad, act), dtype in zip(PADS * 3, ["float32", "bfloat16", "float16", "bfloat16", "float16", "float32", "float16", "float32", "bfloat16"]):
        h, w, hs, ws, bias = _int8_inputs(rows, cin, ctot, M, rows + cin + pad, pad)
        bias = None if act == "linear" else bias
        buf = torch.full((rows, ctot + pad), 55.0, dtype=getattr(torch, dtype), device="cuda:0")
        if groups:
            y = engine.transform_grouped_int8(h, hs, w, ws, ptr, model_of_group=mog, bias=bias, act=act, out=buf[:, :ctot])
        else:
            y = engine.transform_int8(h, hs, w[0], ws[0], bias=None if bias is None else bias[0], act=act, out=buf[:, :ctot])
        of_row = torch.repeat_interleave(torch.tensor(of), torch.tensor([b - a for a, b in blocks])).cuda()
        for m in range(M):
            idx = torch.nonzero(of_row == m).flatten()
            if idx.numel():
                _check_int8_with_overflow(y[idx], h[idx], w[m], hs[idx], ws[m], None if bias is None else bias[m], act, dtype)
        assert bool((buf[:, ctot:] == 55.0).all())


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("rows,cin,ctot,groups", HALF)
def test_half_precision(engine, rows, cin, ctot, groups, dtype):
    import torch
    M, t, g = min(groups, 8), getattr(torch, dtype), _gen(rows + cin)
    ptr, blocks, mog, of = _table(rows, groups)
    of_row = torch.repeat_interleave(torch.tensor(of), torch.tensor([b - a for a, b in blocks])).cuda()
    H, W = torch.randn(rows, cin, device="cuda:0", generator=g).to(t), torch.randn(M, ctot, cin, device="cuda:0", generator=g).to(t)
    bias = torch.randn(M, ctot, device="cuda:0", generator=g)
    for pad, act in PADS:
        b = None if act == "linear" else bias
        buf = torch.full((rows, ctot + pad), 55.0, dtype=t, device="cuda:0")
        y = engine.transform_grouped(_padded(H, pad), W, ptr, model_of_group=mog, bias=b, act=act, out=buf[:, :ctot])
        for m in range(M):
            idx = torch.nonzero(of_row == m).flatten()
            if not idx.numel():
                continue
            h, w = H[idx].double(), W[m].double()
            v, mag = h @ w.t(), h.abs() @ w.abs().t()
            c = b[m].double() if b is not None else torch.zeros(ctot, dtype=torch.float64, device="cuda:0")
            want = _act64(v + c, act)
            tol = 2.01 * U * cin * mag + 2.01 * U * (v.abs() + c.abs())
            tol = tol + HALF_STEP[dtype] * (want.abs() + tol) + SUBNORMAL[dtype]
            assert bool(((y[idx].double() - want).abs() <= tol).all()), (m, act)
        assert bool((buf[:, ctot:] == 55.0).all())


@pytest.mark.parametrize("precise", [False, True])
@pytest.mark.parametrize("rows,cin,ctot,groups", F32)
def test_float32(engine, rows, cin, ctot, groups, precise):
    """Equal bits with ``transform`` under every row's own model."""
    import torch
    M, g = min(groups, 8), _gen(rows + cin)
    ptr, blocks, mog, of = _table(rows, groups)
    H, W = torch.randn(rows, cin, device="cuda:0", generator=g), torch.randn(M, ctot, cin, device="cuda:0", generator=g)
    full = [engine.transform(H, W[m].t().contiguous(), precise=precise) for m in range(M)]
    for pad in (0, 16, 3):
        buf = torch.full((rows, ctot + pad), 55.0, device="cuda:0")
        y = engine.transform_grouped(_padded(H, pad), W, ptr, model_of_group=mog, precise=precise, out=buf[:, :ctot])
        for (lo, hi), m in zip(blocks, of):
            assert torch.equal(y[lo:hi], full[m][lo:hi]), m
        assert bool((buf[:, ctot:] == 55.0).all())
