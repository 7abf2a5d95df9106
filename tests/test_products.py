"""CPU: what the grouped and 8-bit products refuse, at the C entries (no launch happens) and in the Python layer."""
import ctypes as C

import pytest

from distgcn_amd import _lib
from distgcn_amd.engine import Engine, ModelBank

P = 4096  # stands for a device pointer in calls that are refused before anything reads it


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _refused(lib, rc, code, text):
    assert rc == code and text in lib.dgcn_last_error().decode()


def test_quantize_refusals(lib):
    f = lib.dgcn_quantize_rows_batch
    ok = dict(X=P, dtype=0, ldx=8, rows=4, cols=8, Q=P, ldq=8, scale=P, stream=None)
    call = lambda **kw: f(*{**ok, **kw}.values())
    for kw in (dict(X=None), dict(Q=None), dict(scale=None)):
        _refused(lib, call(**kw), -1, "null argument")
    for kw in (dict(rows=-1), dict(cols=0), dict(ldx=7), dict(ldq=7)):
        _refused(lib, call(**kw), -1, "bad sizes")
    _refused(lib, call(dtype=3), -1, "unknown dtype 3")
    assert call(rows=0, X=None, Q=None, scale=None) == 0


def _int8(lib, grouped):
    ok = dict(H=P, ldh=32, hs=P, rows=4, cin=32)
    if grouped:
        ok.update(ptr=P, mog=None, G=2)
    ok.update(W=P, ws=P)
    if grouped:
        ok.update(M=2)
    ok.update(ctot=8, bias=None, act=0, Y=P, dtype=0, ldy=8)
    if grouped:
        ok.update(status=P)
    ok.update(stream=None)
    f = lib.dgcn_transform_grouped_int8_batch if grouped else lib.dgcn_transform_int8_batch
    return lambda **kw: f(*{**ok, **kw}.values())


@pytest.mark.parametrize("grouped", [False, True])
def test_int8_refusals(lib, grouped):
    call = _int8(lib, grouped)
    for k in ("H", "hs", "W", "ws", "Y") + (("ptr", "status") if grouped else ()):
        _refused(lib, call(**{k: None}), -1, "null argument")
    for kw in (dict(rows=-1), dict(cin=0), dict(ctot=0), dict(ldh=31), dict(ldy=7)) + ((dict(G=-1), dict(M=0)) if grouped else ()):
        _refused(lib, call(**kw), -1, "bad sizes")
    _refused(lib, call(dtype=7), -1, "unknown dtype 7")
    _refused(lib, call(act=9), -1, "unknown activation 9")
    _refused(lib, call(cin=131072, ldh=131072), -3, "overflow")
    _refused(lib, call(rows=0x7fffffff), -3, "more than")
    assert call(rows=0) == 0
    if grouped:
        assert call(G=0) == 0


def test_grouped_refusals(lib):
    ok = dict(H=P, dtype=0, ldh=32, const=0.5, rows=4, cin=32, ptr=P, mog=None, G=2, W=P, M=2, ctot=8, bias=None, act=0, precise=0, Y=P,
              ldy=8, status=P, stream=None)
    call = lambda **kw: lib.dgcn_transform_grouped_batch(*{**ok, **kw}.values())
    for k in ("ptr", "W", "Y", "status"):
        _refused(lib, call(**{k: None}), -1, "null argument")
    _refused(lib, call(H=None, dtype=1), -1, "null argument")
    for kw in (dict(rows=-1), dict(cin=0), dict(ctot=0), dict(ldh=31), dict(ldy=7), dict(G=-1), dict(M=0)):
        _refused(lib, call(**kw), -1, "bad sizes")
    _refused(lib, call(dtype=5), -1, "unknown dtype 5")
    _refused(lib, call(act=-1), -1, "unknown activation -1")
    _refused(lib, call(dtype=2, precise=1), -1, "precise takes float32")
    _refused(lib, call(ctot=0x7fffffff, ldy=0x7fffffff), -3, "more than")
    assert call(rows=0) == 0 and call(G=0) == 0


@pytest.fixture()
def host_engine(lib):
    """An Engine whose tensors live in host memory: its argument checks run, a call that passes them all fails the test."""
    import torch
    e = Engine.__new__(Engine)
    e.torch, e.device, e.lib = torch, torch.device("cpu", 0), lib

    def launched(*a):
        raise AssertionError("the arguments were accepted")
    e._launch = launched
    e._here = lambda *a: None
    e._codes = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
    return e


def test_python_refusals(host_engine):
    import torch
    e, z = host_engine, torch.zeros
    H, W, ptr = z(6, 8), z(2, 4, 8), torch.tensor([0, 2, 6], dtype=torch.int32)
    hq, wq, hs, ws = z(6, 8, dtype=torch.int8), z(2, 4, 8, dtype=torch.int8), z(6), z(2, 4)
    with pytest.raises(TypeError):
        e.quantize_rows(z(3, 4, dtype=torch.float64))
    with pytest.raises(ValueError, match="contiguous"):
        e.quantize_rows(z(8, 6).t())
    with pytest.raises(ValueError, match="shape"):
        e.quantize_rows(z(8))
    with pytest.raises(ValueError, match="overlap"):
        e.quantize_rows(z(1, 8).expand(3, 8))
    with pytest.raises(TypeError):
        e.quantize_rows(H, out=(z(6, 8), hs))
    for bad in (dict(H=z(6, 7)), dict(W=z(2, 4, 7)), dict(W=z(4, 8)), dict(bias=z(4)), dict(act="gelu"), dict(out=z(6, 5)),
                dict(group_ptr=z(0, dtype=torch.int32)), dict(W=z(1, 4, 8)), dict(model_of_group=z(3, dtype=torch.int32)),
                dict(status=z(2, dtype=torch.int32)), dict(H=None), dict(H=None, rows=-1), dict(W=z(2, 8, 4).transpose(1, 2)), dict(rows=5)):
        with pytest.raises(ValueError):
            e.transform_grouped(**{**dict(H=H, W=W, group_ptr=ptr), **bad})
    for bad in (dict(H=H.double()), dict(W=W.double(), H=H.double()), dict(H=H.bfloat16()), dict(group_ptr=ptr.long()), dict(out=z(6, 4).half()),
                dict(bias=z(2, 4).half())):
        with pytest.raises(TypeError):
            e.transform_grouped(**{**dict(H=H, W=W, group_ptr=ptr), **bad})
    with pytest.raises(ValueError, match="precise"):
        e.transform_grouped(H.half(), W.half(), ptr, precise=True)
    for bad in (dict(h_scale=z(5)), dict(w_scale=z(4)), dict(Hq=z(6, 9, dtype=torch.int8)), dict(bias=z(4)), dict(act=3)):
        with pytest.raises(ValueError):
            e.transform_grouped_int8(**{**dict(Hq=hq, h_scale=hs, Wq=wq, w_scale=ws, group_ptr=ptr), **bad})
    for bad in (dict(Wq=wq.float()), dict(Hq=hq.float()), dict(dtype=torch.float64), dict(h_scale=hs.double())):
        with pytest.raises(TypeError):
            e.transform_grouped_int8(**{**dict(Hq=hq, h_scale=hs, Wq=wq, w_scale=ws, group_ptr=ptr), **bad})
    for bad in (dict(Wq=wq), dict(w_scale=ws), dict(bias=z(2, 4)), dict(h_scale=z(1)), dict(out=z(5, 4))):
        with pytest.raises(ValueError):
            e.transform_int8(**{**dict(Hq=hq, h_scale=hs, Wq=wq[0], w_scale=ws[0]), **bad})
    with pytest.raises(AssertionError, match="accepted"):
        e.transform_grouped(H, W, ptr)
    with pytest.raises(AssertionError, match="accepted"):
        e.transform_int8(hq, hs, wq[0], ws[0], bias=z(4), act="relu", dtype=torch.bfloat16)


def test_outputs_that_share_memory_are_refused(host_engine):
    import torch
    e = host_engine
    ptr = torch.tensor([0, 2, 6], dtype=torch.int32)
    buf = torch.zeros(6, 24)
    H, W = buf[:, :8], torch.zeros(2, 8, 8)
    for out in (H, buf[:, 4:12], buf.reshape(-1)[:48].reshape(6, 8), buf.reshape(-1)[20:68].reshape(6, 8), W.reshape(16, 8)[3:9]):
        with pytest.raises(ValueError, match="shares memory"):
            e.transform_grouped(H, W, ptr, out=out)
    for out in (buf[:, 8:16], buf[:, 16:], torch.zeros(6, 8)):
        with pytest.raises(AssertionError, match="accepted"):
            e.transform_grouped(H, W, ptr, out=out)
    q = buf.view(torch.int8)
    with pytest.raises(ValueError, match="shares memory"):
        e.quantize_rows(H, out=(q[:, 24:32], torch.zeros(6)))
    with pytest.raises(AssertionError, match="accepted"):
        e.quantize_rows(H, out=(q[:, 32:40], torch.zeros(6)))
    h8 = q[:, :8]
    with pytest.raises(ValueError, match="shares memory"):
        e.transform_int8(h8, torch.zeros(6), torch.zeros(1, 8, dtype=torch.int8), torch.zeros(1), out=buf[:, 1:2])
    with pytest.raises(AssertionError, match="accepted"):
        e.transform_int8(h8, torch.zeros(6), torch.zeros(1, 8, dtype=torch.int8), torch.zeros(1), out=buf[:, 2:3])


def test_rows_beyond_32_bit_offsets_are_refused(lib):
    f, big = lib.dgcn_transform_grouped_batch, 600_000_000  # 2.4 GB of float32 a row
    for dtype, cin in ((0, big), (0, 536870657), (1, 1073741313), (2, 0x7fffffff)):
        rc = f(P, dtype, cin, 0.5, 4, cin, P, None, 2, P, 2, 8, None, 0, 0, P, 8, P, None)
        _refused(lib, rc, -3, "bytes")


def test_bank_refusals(host_engine):
    import numpy as np
    from distgcn_amd import datagen
    e = host_engine
    a, b = datagen.random_model(3, 8, seed=0), datagen.random_model(3, 8, seed=1)
    bank = e.model_bank([a, b])
    assert isinstance(bank, ModelBank) and bank.num_models == 2 and tuple(bank.layers[1]["weights"].shape) == (2, 16, 8)
    assert np.array_equal(bank.layers[1]["weights"][1, 8:].numpy(), b[1]["weights"][1].T)
    for models, kw in (([], {}), ([[]], {}), ([a, datagen.random_model(4, 8)], {}), ([a, datagen.random_model(3, 16)], {}), ([a], dict(precision="int4"))):
        with pytest.raises(ValueError):
            e.model_bank(models, **kw)
    from distgcn_amd.gcn.models import GCN2_DQN, GCN_DQN
    nets = [GCN2_DQN(hidden_dim=8, num_layer=3, input_dim=1, max_degree=1, wts_init="random", seed=s) for s in (1, 2)]
    assert e.model_bank(nets).layers[2]["act"] == "leaky_relu" and e.model_bank(nets, precision="float32").num_models == 2
    with pytest.raises(_lib.DgcnError, match="head"):
        e.model_bank([GCN2_DQN(hidden_dim=8, num_layer=2, input_dim=1, max_degree=1, wts_init="random", output_dim=3, is_dual=True)])
    with pytest.raises(_lib.DgcnError, match="supports"):
        e.model_bank([[dict(lyr, weights=lyr["weights"] + [lyr["weights"][0]]) for lyr in a]])


def test_slots_cover_every_tile_once():
    """The tile arithmetic of the grouped products: group g's row tiles start at slot floor(p_g / BM) + g; the slots of a launch
    (floor(rows / BM) + groups) hold every tile of every group, none twice."""
    import random
    rng = random.Random(5)
    for case in range(300):
        bm = rng.choice([16, 64, 128, 256])
        sizes = [rng.choice([0, 0, 1, bm - 1, bm, bm + 1, rng.randrange(3 * bm)]) for _ in range(rng.randint(1, 40))]
        front, behind = rng.randrange(2 * bm), rng.randrange(2 * bm)
        ptr = [front]
        for s in sizes:
            ptr.append(ptr[-1] + s)
        slots = (ptr[-1] + behind) // bm + len(sizes)
        seen = {}
        for g, s in enumerate(sizes):
            start = ptr[g] // bm + g
            assert g == 0 or start > ptr[g - 1] // bm + g - 1
            for tile in range(-(-s // bm)):
                assert start + tile < slots and start + tile not in seen
                assert g + 1 == len(sizes) or start + tile < ptr[g + 1] // bm + g + 1
                seen[start + tile] = (g, tile)
