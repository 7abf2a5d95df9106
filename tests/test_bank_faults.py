"""CPU: who learns that a batch's supports were made from a faulty adjacency - every call on the batch, not the first alone.

The Engine's device calls are stood in for on the host: the supports launch writes its fault bits, everything else does nothing."""
import ctypes as C

import numpy as np
import pytest

from distgcn_amd import _lib, datagen
from distgcn_amd.batch import DeviceBatch, HostBatch
from distgcn_amd.engine import DeviceModel, Engine

SELF_LOOP = _lib.FAULT_SELF_LOOP


class _Lib:
    """The launches of Engine.supports / supports2 / forward / lgs; `faults` is what the supports kernels would find."""

    def __init__(self, faults):
        self.faults, self.made = faults, 0

    def _word(self, address):
        C.c_int32.from_address(address).value |= self.faults

    def dgcn_supports_batch(self, b, tab, n, row, col, val, status, stream):
        self.made += 1
        self._word(status)
        return 0

    def dgcn_supports2_count_batch(self, b, tab, n, row, status, stream):
        self._word(status)
        return 0

    def dgcn_supports2_fill_batch(self, b, tab, n, row, col, val, status, stream):
        self.made += 1
        self._word(status)
        return 0

    def dgcn_gcn_forward_workspace(self, *a):
        return 256

    def dgcn_gcn_forward_batch(self, *a):
        return 0

    def dgcn_lgs_batch(self, *a):
        return 0

    dgcn_transform_grouped_batch = dgcn_quantize_rows_batch = None  # (never reached: the Engine's _launch is stood in for)


@pytest.fixture()
def host(monkeypatch):
    import torch
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    e = Engine.__new__(Engine)
    e.torch, e.device, e.lib, e._table, e._ws = torch, torch.device("cpu"), _Lib(0), None, None
    e._codes = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
    e._stream, e._index, e._here, e._launch = lambda: None, lambda: -1, lambda *a: None, lambda *a: None
    hb = HostBatch(np.array([0, 2, 5]), np.array([0, 1, 2, 3, 5, 6]), np.array([1, 0, 3, 2, 4, 3]), np.ones(5))
    e.batch = lambda: DeviceBatch(hb, e.device)
    model = datagen.random_model(2, 4, seed=1)
    e.bank, e.model, e.of = e.model_bank([model, model]), DeviceModel(model, "cpu"), torch.zeros(2, dtype=torch.int32)
    e.spmm = lambda lap, Z, out, **kw: torch.zeros(5, out)
    return e


def test_forward_bank_raises_on_every_call(host):
    host.lib.faults = SELF_LOOP
    b = host.batch()
    for _ in range(3):
        with pytest.raises(_lib.DgcnError, match="self-loop"):
            host.forward_bank(b, host.bank, host.of)
    with pytest.raises(_lib.DgcnError, match="self-loop"):
        host.forward(b, host.model)
    with pytest.raises(_lib.DgcnError, match="self-loop"):
        host.supports(b)


def test_a_caller_s_word_gets_the_faults_every_time(host):
    import torch
    host.lib.faults = SELF_LOOP
    b = host.batch()
    for _ in range(3):
        word = torch.zeros(1, dtype=torch.int32)
        host.forward_bank(b, host.bank, host.of, status=word)
        assert int(word) == SELF_LOOP
        assert int(host.solve_bank(b, host.bank, host.of)["status"]) == SELF_LOOP
        assert int(host.solve(b, host.model)["status"]) == SELF_LOOP
    with pytest.raises(_lib.DgcnError, match="self-loop"):
        host.forward_bank(b, host.bank, host.of)
    with pytest.raises(_lib.DgcnError, match="self-loop"):
        host.forward(b, host.model)


def test_the_faults_are_the_batch_s_own(host):
    """What else is in a caller's word does not become a fault of the batch, and a word the caller clears takes nothing back."""
    import torch
    b = host.batch()
    word = torch.full((1,), _lib.FAULT_NAN_PRIORITY, dtype=torch.int32)
    host.supports(b, status=word)
    assert int(word) == _lib.FAULT_NAN_PRIORITY
    res = host.solve(b, host.model)
    res["status"].fill_(_lib.FAULT_NAN_PRIORITY)
    assert int(host.solve(b, host.model)["status"]) == 0 and host.lib.made == 1
    host.forward_bank(b, host.bank, host.of)
    host.forward(b, host.model)
    host.lib.faults = SELF_LOOP
    bad = host.batch()
    word.zero_()
    host.supports(bad, status=word)
    word.zero_()
    assert int(host.solve(bad, host.model)["status"]) == SELF_LOOP
    host.supports(b, status=word)
    assert int(word) == 0
    bad.lap = None  # made anew, by an adjacency without fault
    host.lib.faults = 0
    assert int(host.solve(bad, host.model)["status"]) == 0


def test_second_supports_keep_their_faults(host):
    import torch
    host.lib.faults = _lib.FAULT_BAD_COLUMN
    b = host.batch()
    for _ in range(2):
        word = torch.zeros(1, dtype=torch.int32)
        host.supports2(b, status=word)
        assert int(word) == _lib.FAULT_BAD_COLUMN
    for _ in range(2):
        with pytest.raises(_lib.DgcnError, match="column"):
            host.supports2(b)


def test_supports_from_elsewhere_have_no_faults(host):
    b = host.batch()
    host.supports(b)
    b.lap = {k: v for k, v in b.lap.items() if k in ("row_ptr", "col_idx", "values", "c")}  # as a feed's own supports are set
    assert int(host.solve(b, host.model)["status"]) == 0
    host.forward(b, host.model)
    host.forward_bank(b, host.bank, host.of)


def test_an_8_bit_layer_keeps_one_form_of_its_weights(host):
    models = [datagen.random_model(3, 4, seed=s) for s in (1, 2)]
    first, hidden, last = host.model_bank(models, precision="int8").layers
    assert hidden["weights"] is None and tuple(hidden["q"].shape) == (2, 8, 4) and tuple(hidden["scale"].shape) == (2, 8)
    for layer in (first, last):
        assert layer["weights"] is not None and layer["q"] is None and layer["scale"] is None


@pytest.fixture()
def checks():
    """An Engine on the host whose argument checks run; a call that passes them all raises AssertionError("accepted")."""
    import torch
    e = Engine.__new__(Engine)
    e.torch, e.device, e.lib = torch, torch.device("cpu"), _lib.load()
    e._codes = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
    e._here = lambda *a: None

    def launched(*a):
        raise AssertionError("accepted")
    e._launch = launched
    return e


def _refused(call, **kw):
    with pytest.raises(ValueError, match="shares memory"):
        call(**kw)


def _taken(call, **kw):
    with pytest.raises(AssertionError, match="accepted"):
        call(**kw)


def test_outputs_apart_from_scales_biases_and_tables(checks):
    import torch
    e = checks
    buf = torch.zeros(64 * 16)
    at = lambda lo, *shape: buf[lo:lo + int(np.prod(shape))].view(*shape)
    ints = lambda lo, n: at(lo, n).view(torch.int32)
    out = at(256, 8, 16)[:, :10]  # elements 256 .. 383, six free ones behind each row's ten
    H, W = torch.zeros(8, 4), torch.zeros(2, 10, 4)
    h8, w8 = torch.zeros(8, 4, dtype=torch.int8), torch.zeros(2, 10, 4, dtype=torch.int8)
    ptr, mog, word = torch.tensor([0, 3, 8], dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    hs, ws, bias = torch.zeros(8), torch.zeros(2, 10), torch.zeros(2, 10)
    f = lambda **kw: e.transform_grouped(**{**dict(H=H, W=W, group_ptr=ptr, model_of_group=mog, bias=bias, out=out, status=word), **kw})
    g = lambda **kw: e.transform_grouped_int8(**{**dict(Hq=h8, h_scale=hs, Wq=w8, w_scale=ws, group_ptr=ptr, model_of_group=mog, bias=bias, out=out, status=word), **kw})
    d = lambda **kw: e.transform_int8(**{**dict(Hq=h8, h_scale=hs, Wq=w8[0], w_scale=ws[0], bias=bias[0], out=out), **kw})
    for call in (f, g):
        _taken(call)
        for lo in (256 - 19, 256, 262, 266, 276, 383 - 16 - 6):  # into the first row, over it, from a gap into the next row, the last row
            _refused(call, bias=at(lo, 2, 10))
        _taken(call, bias=at(256 - 20, 2, 10))
        _taken(call, bias=at(378, 2, 10))  # behind the last row's ten
        _refused(call, group_ptr=ints(256 + 32 + 8, 3))
        _taken(call, group_ptr=ints(256 + 32 + 10, 3))  # a gap
        _refused(call, group_ptr=ints(256 + 32 + 14, 3))
        _refused(call, model_of_group=ints(256 + 9, 2))
        _refused(call, status=ints(256 + 48, 1))
        _taken(call, status=ints(256 + 48 - 1, 1))
    _taken(g, h_scale=at(0, 8), w_scale=at(8, 2, 10))
    _refused(g, h_scale=at(250, 8))
    _refused(g, w_scale=at(370, 2, 10))
    _taken(d)
    _refused(d, h_scale=at(250, 8))
    _refused(d, w_scale=at(250, 10))
    _refused(d, bias=at(270, 10))
    X, q = at(256, 8, 16)[:, :10], at(512, 8, 16).view(torch.int8)[:, :10]
    qz = lambda scale: e.quantize_rows(X, out=(q, scale))
    _taken(qz, scale=at(0, 8))
    _taken(qz, scale=at(512 - 8, 8))
    for lo in (250, 300, 376, 505, 512, 521):
        _refused(qz, scale=at(lo, 8))
    _taken(qz, scale=at(512 + 16 * 3 + 3, 8))  # q's rows take 10 bytes of 64


def test_empty_outputs_share_nothing(checks):
    import torch
    e, z = checks, torch.zeros
    buf = z(100)
    _taken(e.transform_grouped, H=z(0, 4), W=z(1, 10, 4), group_ptr=torch.zeros(2, dtype=torch.int32), bias=buf[:10].view(1, 10), out=buf[:0].view(0, 10),
           status=torch.zeros(1, dtype=torch.int32))
    _taken(e.quantize_rows, X=z(0, 4), out=(z(0, 4, dtype=torch.int8), z(0)))


def test_sizes_beyond_32_bits_are_refused(checks):
    """They reach the library as 32-bit numbers: 2^32 + 5 rows would be five."""
    import torch
    e, big = checks, 2 ** 32 + 5
    m = lambda *shape, **kw: torch.empty(*shape, device="meta", **kw)
    i8 = dict(dtype=torch.int8)
    word, ptr = torch.zeros(1, dtype=torch.int32), torch.tensor([0, 4], dtype=torch.int32)
    calls = [lambda: e.quantize_rows(m(big, 1)), lambda: e.quantize_rows(m(1, big)), lambda: e.quantize_rows(m(3, big, dtype=torch.float16)),
             lambda: e.transform_int8(m(big, 4, **i8), m(big), m(3, 4, **i8), m(3)), lambda: e.transform_int8(m(2, big, **i8), m(2), m(3, big, **i8), m(3)),
             lambda: e.transform_int8(m(2, 4, **i8), m(2), m(big, 4, **i8), m(big)),
             lambda: e.transform_grouped(m(big, 4), m(1, 3, 4), ptr, status=word), lambda: e.transform_grouped(m(4, 4), m(big, 3, 4), ptr, status=word),
             lambda: e.transform_grouped(m(4, 4), m(1, big, 4), ptr, status=word), lambda: e.transform_grouped(None, m(1, 3, 4), ptr, rows=big, status=word),
             lambda: e.transform_grouped(None, m(1, 3, big), ptr, rows=4, status=word),
             lambda: e.transform_grouped(m(4, 4), m(1, 3, 4), m(big + 1, dtype=torch.int32), model_of_group=m(big, dtype=torch.int32), status=word),
             lambda: e.transform_grouped_int8(m(big, 4, **i8), m(big), m(1, 3, 4, **i8), m(1, 3), ptr, status=word)]
    for i, call in enumerate(calls):
        with pytest.raises(ValueError, match="32 bits"):
            call()
