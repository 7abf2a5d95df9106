"""Device engine: thin Python over the C ABI (include/dgcn.h).

PyTorch is used for device memory and streams only; every computation on the path runs in
libdgcn.so.  All methods enqueue on the current torch stream and do not synchronise unless they
return host data.
"""
from __future__ import annotations

import ctypes as C
import os
from typing import List, Optional

import numpy as np

from . import _lib
from .batch import DeviceBatch, HostBatch

ACT_CODES = {"linear": _lib.ACT_LINEAR, "identity": _lib.ACT_LINEAR, None: _lib.ACT_LINEAR,
             "leaky_relu": _lib.ACT_LEAKY_RELU, "relu": _lib.ACT_RELU}

MODE_LAYERED, MODE_FUSED = 0, 1


def dinv_table(max_degree: int) -> np.ndarray:
    """float64 d^-1/2 for d = 0..max_degree with inf -> 0, computed with the very NumPy call the
    reference uses (gcn/utils.py:124-125) so the bits agree."""
    d = np.arange(max_degree + 1, dtype=np.float64)
    with np.errstate(divide="ignore"):
        t = np.power(d, -0.5)
    t[np.isinf(t)] = 0.0
    return t


_NP = {"uint8": np.uint8, "int32": np.int32, "int64": np.int64, "float32": np.float32, "float64": np.float64}


def packed_layout(specs):
    """(total bytes, {name: (byte offset, bytes, dtype name)}) of arrays packed into one byte buffer, widest
    element type first, every array 16-byte aligned.  specs: (name, element count, dtype name); count 0 = absent."""
    off, lay = 0, {}
    for name, count, dt in sorted(specs, key=lambda x: -np.dtype(_NP[x[2]]).itemsize):
        if count <= 0:
            continue
        nb = count * np.dtype(_NP[dt]).itemsize
        lay[name] = (off, nb, dt)
        off = (off + nb + 15) & ~15
    return max(off, 16), lay


def solve_buffer_specs(num_nodes: int, num_graphs: int, want_scores: bool):
    """The arrays of one rank's packed solve result (``Engine.solve_buffers``)."""
    return [("totals", num_graphs, "float64"), ("scores", num_nodes if want_scores else 0, "float32"),
            ("rounds", num_graphs, "int32"), ("status", 1, "int32"), ("state", num_nodes, "uint8")]


class DeviceModel:
    """Layer stack on the device.  ``layers`` is a list of dicts
    {"weights": [W_0, W_1] (each [in, out] float32), "bias": None | [out], "act": str}."""

    def __init__(self, layers: List[dict], device="cuda"):
        import torch
        if not layers:
            raise ValueError("model has no layers")
        self.device = torch.device(device)
        self.layers = layers
        self.num_supports = len(layers[0]["weights"])
        self._keep = []
        arr = (_lib.DgcnLayer * len(layers))()
        for i, lyr in enumerate(layers):
            ws = [np.asarray(w, dtype=np.float32) for w in lyr["weights"]]
            if len(ws) != self.num_supports:
                raise ValueError("layer %d has %d weight matrices, expected %d" % (i, len(ws), self.num_supports))
            cat = np.ascontiguousarray(np.concatenate(ws, axis=1))  # [in, K*out]
            wt = torch.from_numpy(cat).to(self.device)
            bt = None
            if lyr.get("bias") is not None:
                bt = torch.from_numpy(np.ascontiguousarray(lyr["bias"], dtype=np.float32).ravel()).to(self.device)
            self._keep += [wt, bt]
            arr[i] = _lib.DgcnLayer(ws[0].shape[0], ws[0].shape[1], wt.data_ptr(),
                                    bt.data_ptr() if bt is not None else None, ACT_CODES[lyr.get("act")])
        self._layer_arr = arr
        self.c = _lib.DgcnModel(len(layers), self.num_supports, arr)
        self.in_dim = int(arr[0].in_dim)
        self.out_dim = int(arr[len(layers) - 1].out_dim)


class ModelBank:
    """Several models of one architecture on the device, for batches whose graphs belong to different models
    (``Engine.forward_bank`` / ``solve_bank``; ``Engine.model_bank`` makes one).  ``layers`` = per layer {"weights": float32
    [models, 2 * out, in] (both supports' weights, an output column's weights contiguous) or None where the 8-bit form stands for them,
    "bias": None | float32 [models, 2 * out] (0 behind the first half), "act", "in", "out", "q" / "scale": the 8-bit form or None}."""

    def __init__(self, layers, num_models: int, precision: str):
        self.layers, self.num_models, self.precision = layers, num_models, precision
        self.in_dim, self.out_dim = layers[0]["in"], layers[-1]["out"]


def _matrix(x, what, dtypes, cols=None, rows=None):
    """Check a 2-D tensor whose rows are contiguous; -> (rows, columns, row stride in elements)."""
    if x.dtype not in dtypes:
        raise TypeError("%s is %s, expected %s" % (what, x.dtype, " / ".join(str(d) for d in dtypes)))
    shape = x.shape
    if len(shape) != 2 or (cols is not None and shape[1] != cols) or (rows is not None and shape[0] != rows):
        raise ValueError("%s has shape %s, expected [%s, %s]" % (what, tuple(shape), "rows" if rows is None else rows,
                                                                 "columns" if cols is None else cols))
    r, c = shape
    ld, inner = x.stride()
    if inner != 1 and c > 1:
        raise ValueError("%s: the entries of a row must be contiguous" % what)
    if r <= 1:
        return r, c, max(c, 1)
    if ld < c:
        raise ValueError("%s: rows overlap (row stride %d, %d columns)" % (what, ld, c))
    return r, c, ld


def _overlap(x, ldx, y, ldy):
    """Do two matrices share memory?  Column ranges of one buffer's rows do not."""
    ax, ay, ex, ey = x.data_ptr(), y.data_ptr(), x.element_size(), y.element_size()
    r, c = x.shape[-2:]
    if x.dim() == 3:
        r *= x.shape[0]
    s, d = y.shape
    if ax + ((r - 1) * ldx + c) * ex <= ay or ay + ((s - 1) * ldy + d) * ey <= ax or not r or not s:
        return False
    pitch = ldx * ex
    off = (ay - ax) % max(pitch, 1)
    return pitch != ldy * ey or off < c * ex or off + d * ey > pitch


def _apart(y, ldy, what, *arrays):
    """Refuse contiguous tensors of 32-bit numbers (None: not given) that share memory with a matrix; what lies between its rows is not
    part of it."""
    rows, cols = y.shape
    start, size = y.data_ptr(), y.element_size()
    end = start + ((rows - 1) * ldy + cols) * size
    for x in arrays:
        if x is None:
            continue
        lo = x.data_ptr()
        if lo >= end:
            continue
        hi = lo + 4 * x.numel()
        if hi <= start or lo == hi or not rows or not cols:
            continue
        at, pitch = max(lo - start, 0), ldy * size
        if at % pitch < cols * size or hi - start > (at // pitch + 1) * pitch:
            raise ValueError("%s shares memory with another argument" % what)


def _array(x, what, dtype, shape):
    """Check a contiguous tensor of one dtype and shape."""
    if x.dtype != dtype:
        raise TypeError("%s is %s, expected %s" % (what, x.dtype, dtype))
    if x.shape != shape:
        raise ValueError("%s has shape %s, expected %s" % (what, tuple(x.shape), shape))
    if not x.is_contiguous():
        raise ValueError("%s must be contiguous" % what)


class Engine:
    def __init__(self, device="cuda"):
        import torch
        if not torch.cuda.is_available():
            raise _lib.DgcnError("no GPU visible: distgcn_amd runs on MI355X only (there is no CPU fallback)")
        self.torch = torch
        self.device = torch.device(device)
        self.lib = _lib.load()
        self._table = None
        self._ws = None
        self._codes = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}  # the products' floating-point types
        raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # (the same handle without building a Stream object)
        self._raw_stream = raw or (lambda index: torch.cuda.current_stream(index).cuda_stream)

    # ------------------------------------------------------------------ helpers
    def _stream(self):
        return C.c_void_p(self.torch.cuda.current_stream(self.device).cuda_stream)

    def _dinv(self, max_degree: int):
        if self._table is None or self._table.numel() <= max_degree:
            n = max(1024, 2 * (max_degree + 1))
            self._table = self.torch.from_numpy(dinv_table(n - 1)).to(self.device)
        return self._table

    def _workspace(self, nbytes: int):
        if self._ws is None or self._ws.numel() < nbytes:
            self._ws = self.torch.empty(max(nbytes, 256), dtype=self.torch.uint8, device=self.device)
        return self._ws

    _NP = _NP

    def _packed(self, specs):
        """Device arrays as views into ONE byte tensor, so a caller can fetch them all with a single
        device-to-host copy (``fetch_packed``).  specs: (name, element count, dtype name); count 0 = absent."""
        t = self.torch
        off, lay = packed_layout(specs)
        flat = t.zeros(off, dtype=t.uint8, device=self.device)
        out = {"flat": flat, "layout": lay}
        for name, _, _ in specs:
            if name in lay:
                o, nb, dt = lay[name]
                out[name] = flat[o:o + nb].view(getattr(t, dt))
            else:
                out[name] = None
        return out

    @classmethod
    def fetch_packed(cls, out):
        """One device-to-host copy -> {name: NumPy array} for everything ``_packed`` laid out."""
        host = out["flat"].cpu().numpy()
        return {name: host[o:o + nb].view(cls._NP[dt]) for name, (o, nb, dt) in out["layout"].items()}

    def upload(self, host: HostBatch) -> DeviceBatch:
        with self.torch.cuda.device(self.device):
            return DeviceBatch(host, self.device)

    def check_status(self, status) -> None:
        self.check_status_bits(int(status.item()))

    @staticmethod
    def check_status_bits(bits: int) -> None:
        if bits & 16:
            # the cluster variant of the fused kernel relies on a placement that this device / partition mode does not give:
            # switch it off for the rest of the process, so that a retry (and every later call) takes the ordinary launch
            _lib.load().dgcn_set_cluster(0)
        if bits:
            raise _lib.DgcnError("device-side validation failed: " + _lib.fault_text(bits))

    # ------------------------------------------------------------------ A1/A2
    def supports(self, b: DeviceBatch, status=None):
        """L = I - D^-1/2 A D^-1/2 for the batch (gcn/utils.py:258-274, k=1).  Made once and kept with the batch, with the faults of its
        adjacency: every call ORs them into ``status``, or raises without one (a call in a stream capture cannot: read
        the word of the call that made them)."""
        if b.lap is None:
            lap = self._make_supports(b)
            if status is None:
                self.check_status(lap["faults"])
                lap["checked"] = True
            b.lap = lap
        return self._kept(b.lap, status)

    def _make_supports(self, b: DeviceBatch):
        t = self.torch
        n, e = b.host.num_nodes, b.host.num_edges
        row_ptr = t.empty(n + 1, dtype=t.int32, device=self.device)
        col = t.empty(max(n + e, 1), dtype=t.int32, device=self.device)
        val = t.empty(max(n + e, 1), dtype=t.float32, device=self.device)
        faults = t.zeros(1, dtype=t.int32, device=self.device)
        tab = self._dinv(b.host.max_degree)
        if n == 0:
            row_ptr.zero_()
        _lib.check(self.lib.dgcn_supports_batch(C.byref(b.c), tab.data_ptr(), int(tab.numel()), row_ptr.data_ptr(),
                                                col.data_ptr(), val.data_ptr(), faults.data_ptr(), self._stream()),
                   "dgcn_supports_batch")
        csr = _lib.DgcnCsr(n, n + e, b.host.max_graph_edges + b.host.max_nodes, row_ptr.data_ptr(), col.data_ptr(), val.data_ptr())
        return {"row_ptr": row_ptr, "col_idx": col, "values": val, "c": csr, "faults": faults, "checked": False}

    def _kept(self, made, status):
        """A batch's kept supports for one more call.  "faults": the word their kernel wrote (None or absent: supports from elsewhere);
        "checked": the host has read it and it is 0.  (The word stays with them: a captured call may read it again.)"""
        if made.get("faults") is not None and not made["checked"]:
            if status is not None:
                status.bitwise_or_(made["faults"])
            elif not self.torch.cuda.is_current_stream_capturing():
                self.check_status(made["faults"])
                made["checked"] = True
        return made

    def _call_status(self, b: DeviceBatch):
        """A status word for one call on the batch, the faults of its supports in it; makes the supports if need be."""
        t = self.torch
        if b.lap is None:
            b.lap = self._make_supports(b)
        if b.lap.get("faults") is None or b.lap["checked"]:
            return t.zeros(1, dtype=t.int32, device=self.device)
        return b.lap["faults"] + 0

    def supports2(self, b: DeviceBatch, status=None):
        """T_2 = L.L for the batch, formed explicitly like the reference's ``t_k[-1]*laplacian``
        (gcn/utils.py:268-271); float32 values bit-identical to the reference's.  Kept with the batch, its faults too (``supports``).
        One device-to-host read of the entry count between the two passes (the caller allocates)."""
        t = self.torch
        if getattr(b, "lap2", None) is not None:
            return self._kept(b.lap2, status)
        n = b.host.num_nodes
        faults = t.zeros(1, dtype=t.int32, device=self.device)
        tab = self._dinv(b.host.max_degree)
        row_ptr = t.zeros(n + 1, dtype=t.int32, device=self.device)
        _lib.check(self.lib.dgcn_supports2_count_batch(C.byref(b.c), tab.data_ptr(), int(tab.numel()), row_ptr.data_ptr(),
                                                       faults.data_ptr(), self._stream()), "dgcn_supports2_count_batch")
        nnz = int(row_ptr[n].item())
        col = t.empty(max(nnz, 1), dtype=t.int32, device=self.device)
        val = t.empty(max(nnz, 1), dtype=t.float32, device=self.device)
        _lib.check(self.lib.dgcn_supports2_fill_batch(C.byref(b.c), tab.data_ptr(), int(tab.numel()), row_ptr.data_ptr(),
                                                      col.data_ptr(), val.data_ptr(), faults.data_ptr(), self._stream()),
                   "dgcn_supports2_fill_batch")
        if status is None:
            self.check_status(faults)
        csr = _lib.DgcnCsr(n, nnz, 0, row_ptr.data_ptr(), col.data_ptr(), val.data_ptr())
        b.lap2 = {"row_ptr": row_ptr, "col_idx": col, "values": val, "c": csr, "faults": faults, "checked": status is None}
        return self._kept(b.lap2, status)

    # ------------------------------------------------------------------ K4
    def spmm(self, csr: dict, Z, C_feat: int, ldz: Optional[int] = None, graph_ptr=None, num_graphs=0, max_nodes=0,
             Y0=None, ldy0=0, bias=None, act="linear", out=None, precise=False):
        """``precise``: the row sums carried in double (``dgcn_spmm_f64acc_batch``, the contract of layer index 0)."""
        t = self.torch
        n = int(csr["c"].num_rows)
        ldz = ldz or int(Z.shape[-1])
        if out is None:
            out = t.empty((n, C_feat), dtype=t.float32, device=self.device)
        if precise:
            _lib.check(self.lib.dgcn_spmm_f64acc_batch(
                C.byref(csr["c"]), graph_ptr.data_ptr() if graph_ptr is not None else None, num_graphs, max_nodes,
                Z.data_ptr(), ldz, C_feat, Y0.data_ptr() if Y0 is not None else None, ldy0,
                bias.data_ptr() if bias is not None else None, ACT_CODES[act], out.data_ptr(), int(out.shape[-1]),
                self._stream()), "dgcn_spmm_f64acc_batch")
            return out
        _lib.check(self.lib.dgcn_spmm_batch(
            C.byref(csr["c"]), graph_ptr.data_ptr() if graph_ptr is not None else None, num_graphs, max_nodes,
            Z.data_ptr(), ldz, C_feat, Y0.data_ptr() if Y0 is not None else None, ldy0,
            bias.data_ptr() if bias is not None else None, ACT_CODES[act], out.data_ptr(), int(out.shape[-1]),
            self._stream()), "dgcn_spmm_batch")
        return out

    # ------------------------------------------------------------------ K2/K3
    def transform(self, H, W, rows: Optional[int] = None, h_const: float = 1.0, precise=False):
        """``precise``: the k chains carried in double (``dgcn_transform_f64acc_batch``, the contract of layer index 1)."""
        t = self.torch
        cin, ctot = int(W.shape[0]), int(W.shape[1])
        if H is not None:
            rows = int(H.shape[0])
        out = t.empty((rows, ctot), dtype=t.float32, device=self.device)
        fn = self.lib.dgcn_transform_f64acc_batch if precise else self.lib.dgcn_transform_batch
        _lib.check(fn(H.data_ptr() if H is not None else None,
                                                 int(H.shape[1]) if H is not None else cin, h_const, rows, cin,
                                                 W.data_ptr(), ctot, out.data_ptr(), ctot, self._stream()),
                   "dgcn_transform_batch")
        return out

    # ------------------------------------------------------------------ K2/K3 for several models / in 8-bit integers
    def _index(self):
        """Number of this engine's device."""
        index = self.device.index
        return self.torch.cuda.current_device() if index is None else index

    def _here(self, *tensors):
        """Every tensor (None: not given) lives on this engine's device."""
        index = self._index()
        for x in tensors:
            if x is not None and x.get_device() != index:
                raise ValueError("a tensor is on %s, the engine on %s" % (x.device, self.device))

    def _launch(self, fn, what, *args):
        """One library call on this engine's device and its current stream."""
        index = self._index()
        if index == self.torch.cuda.current_device():
            rc = fn(*args, self._raw_stream(index))
        else:
            with self.torch.cuda.device(index):
                rc = fn(*args, self._raw_stream(index))
        if rc:
            _lib.check(rc, what)

    def _product_args(self, H, W, bias, act, dtype, out, grouped, rows=None):
        """The checks every product shares, but for the device -> (rows, cin, ctot, models, ldh, activation code, dtype code, out, ldy)."""
        codes = self._codes
        if dtype not in codes:
            raise TypeError("dtype is %s, expected %s" % (dtype, " / ".join(str(d) for d in codes)))
        if act not in ACT_CODES:
            raise ValueError("unknown activation %r" % (act,))
        shape = W.shape
        if len(shape) != (3 if grouped else 2):
            raise ValueError("the weights have shape %s, expected %s" % (tuple(shape), "[models, ctot, cin]" if grouped else "[ctot, cin]"))
        if not W.is_contiguous():
            raise ValueError("the weights must be contiguous")
        M, ctot, cin = shape if grouped else (1, *shape)
        ldh = cin
        if H is not None:
            rows, _, ldh = _matrix(H, "H", (W.dtype,), cols=cin, rows=rows)
        if (rows | M | ctot | cin) >> 31:
            raise ValueError("weights of shape %s, %d rows: sizes are numbers of 32 bits" % (tuple(shape), rows))
        if bias is not None:
            _array(bias, "bias", self.torch.float32, (M, ctot) if grouped else (ctot,))
        if out is None:
            out, ldy = self.torch.empty((rows, ctot), dtype=dtype, device=self.device), max(ctot, 1)
        else:
            ldy = _matrix(out, "out", (dtype,), cols=ctot, rows=rows)[2]
            if (H is not None and _overlap(H, ldh, out, ldy)) or _overlap(W, cin, out, ldy):
                raise ValueError("out shares memory with H or the weights")
        return rows, cin, ctot, M, ldh, ACT_CODES[act], codes[dtype], out, ldy

    def _groups(self, group_ptr, model_of_group, num_models, status):
        """The arguments every grouped product shares -> (number of groups, status word, is the word this call's own)."""
        t = self.torch
        shape = group_ptr.shape
        if len(shape) != 1 or shape[0] < 1:
            raise ValueError("group_ptr has shape %s, expected [groups + 1]" % (tuple(shape),))
        G = shape[0] - 1
        if G >> 31:
            raise ValueError("%d groups: their number has 32 bits" % G)
        _array(group_ptr, "group_ptr", t.int32, shape)
        if model_of_group is not None:
            _array(model_of_group, "model_of_group", t.int32, (G,))
        elif num_models < G:
            raise ValueError("%d groups but %d models (and no model_of_group)" % (G, num_models))
        own = status is None
        if own:
            status = t.zeros(1, dtype=t.int32, device=self.device)
        else:
            _array(status, "status", t.int32, (1,))
        self._here(group_ptr, model_of_group, status)
        return G, status, own

    def quantize_rows(self, X, out=None):
        """Dynamic 8-bit quantisation of the rows of X (float32 / bfloat16 / float16, any row stride):
        ``q = X / scale`` rounded half to even, ``scale = max|row| / 127`` (``dgcn_quantize_rows_batch``).  The same call
        quantises weights, a row per output column.  ``out = (q, scale)`` re-uses buffers.  -> (int8 [rows, cols], float32 [rows]);
        a row with a NaN or an infinity gets scale NaN."""
        t = self.torch
        codes = self._codes
        rows, cols, ldx = _matrix(X, "X", codes)
        if (rows | cols) >> 31:
            raise ValueError("X has shape %s: rows and columns are numbers of 32 bits" % (tuple(X.shape),))
        if out is None:
            q, scale = t.empty((rows, cols), dtype=t.int8, device=self.device), t.empty(rows, dtype=t.float32, device=self.device)
            ldq = max(cols, 1)
        else:
            q, scale = out
            ldq = _matrix(q, "q", (t.int8,), cols=cols, rows=rows)[2]
            if _overlap(X, ldx, q, ldq):
                raise ValueError("q shares memory with X")
            _array(scale, "scale", t.float32, (rows,))
            _apart(X, ldx, "X", scale)
            _apart(q, ldq, "q", scale)
        self._here(X, q, scale)
        self._launch(self.lib.dgcn_quantize_rows_batch, "dgcn_quantize_rows_batch", X.data_ptr(), codes[X.dtype], ldx, rows, cols,
                     q.data_ptr(), ldq, scale.data_ptr())
        return q, scale

    def transform_int8(self, Hq, h_scale, Wq, w_scale, bias=None, act="linear", dtype=None, out=None):
        """``act((Hq . Wq^T) * h_scale * w_scale + bias)`` (``dgcn_transform_int8_batch``): Hq int8 [rows, cin] with a scale per row,
        Wq int8 [ctot, cin] (an output column's weights contiguous) with a scale per output column; exact int32 sums, float32 behind
        them, ``dtype`` (float32 / bfloat16 / float16) out."""
        t = self.torch
        if Wq.dtype != t.int8:
            raise TypeError("Wq is %s, expected torch.int8" % Wq.dtype)
        given = out is not None
        rows, cin, ctot, _, ldh, code, dt, out, ldy = self._product_args(
            Hq, Wq, bias, act, dtype or (t.float32 if out is None else out.dtype), out, False)
        _array(h_scale, "h_scale", t.float32, (rows,))
        _array(w_scale, "w_scale", t.float32, (ctot,))
        if given:
            _apart(out, ldy, "out", h_scale, w_scale, bias)
        self._here(Hq, Wq, h_scale, w_scale, bias, out)
        self._launch(self.lib.dgcn_transform_int8_batch, "dgcn_transform_int8_batch", Hq.data_ptr(), ldh, h_scale.data_ptr(), rows, cin,
                     Wq.data_ptr(), w_scale.data_ptr(), ctot, None if bias is None else bias.data_ptr(), code, out.data_ptr(), dt, ldy)
        return out

    def transform_grouped(self, H, W, group_ptr, model_of_group=None, bias=None, act="linear", rows: Optional[int] = None,
                          h_const: float = 1.0, precise=False, out=None, status=None):
        """``act(H . W[m]^T + bias[m])``, m the model of the row's group (``dgcn_transform_grouped_batch``): group g owns the rows
        ``group_ptr[g] .. group_ptr[g + 1]`` (int32 on the device, e.g. a batch's ``graph_ptr``) and takes model
        ``model_of_group[g]`` (None: model g).  W is [models, ctot, cin] (an output column's weights contiguous), H float32 /
        bfloat16 / float16 like W, or None for float32 features that all equal ``h_const`` (``rows`` of them).  float32: the bits of
        ``transform`` with the row's model; ``precise`` as there.  Rows outside every group are left as they were: what ``out``
        held, nothing defined in a result made here.  With ``status`` (an int32 word the caller zeroed) nothing waits and faults are the
        caller's to read; without, they raise here."""
        t = self.torch
        if H is None and (W.dtype != t.float32 or rows is None or rows < 0):
            raise ValueError("constant features need float32 weights and the number of rows")
        if precise and W.dtype != t.float32:
            raise ValueError("precise takes float32")
        given = out is not None
        rows, cin, ctot, M, ldh, code, dt, out, ldy = self._product_args(H, W, bias, act, W.dtype, out, True, rows)
        self._here(H, W, bias, out)
        G, status, own = self._groups(group_ptr, model_of_group, M, status)
        if given:
            _apart(out, ldy, "out", bias, group_ptr, model_of_group, status)
        self._launch(self.lib.dgcn_transform_grouped_batch, "dgcn_transform_grouped_batch", None if H is None else H.data_ptr(), dt, ldh,
                     float(h_const), rows, cin, group_ptr.data_ptr(), None if model_of_group is None else model_of_group.data_ptr(), G,
                     W.data_ptr(), M, ctot, None if bias is None else bias.data_ptr(), code, 1 if precise else 0, out.data_ptr(), ldy,
                     status.data_ptr())
        if own:
            self.check_status(status)
        return out

    def transform_grouped_int8(self, Hq, h_scale, Wq, w_scale, group_ptr, model_of_group=None, bias=None, act="linear", dtype=None,
                               out=None, status=None):
        """``transform_int8`` with Wq [models, ctot, cin], w_scale and bias [models, ctot] of the row's model; groups and ``status`` as in
        ``transform_grouped`` (``dgcn_transform_grouped_int8_batch``)."""
        t = self.torch
        if Wq.dtype != t.int8:
            raise TypeError("Wq is %s, expected torch.int8" % Wq.dtype)
        given = out is not None
        rows, cin, ctot, M, ldh, code, dt, out, ldy = self._product_args(
            Hq, Wq, bias, act, dtype or (t.float32 if out is None else out.dtype), out, True)
        _array(h_scale, "h_scale", t.float32, (rows,))
        _array(w_scale, "w_scale", t.float32, (M, ctot))
        self._here(Hq, Wq, h_scale, w_scale, bias, out)
        G, status, own = self._groups(group_ptr, model_of_group, M, status)
        if given:
            _apart(out, ldy, "out", h_scale, w_scale, bias, group_ptr, model_of_group, status)
        self._launch(self.lib.dgcn_transform_grouped_int8_batch, "dgcn_transform_grouped_int8_batch", Hq.data_ptr(), ldh,
                     h_scale.data_ptr(), rows, cin, group_ptr.data_ptr(), None if model_of_group is None else model_of_group.data_ptr(), G,
                     Wq.data_ptr(), w_scale.data_ptr(), M, ctot, None if bias is None else bias.data_ptr(), code, out.data_ptr(), dt, ldy,
                     status.data_ptr())
        if own:
            self.check_status(status)
        return out

    # ------------------------------------------------------------------ A4-A6
    def forward(self, b: DeviceBatch, model: DeviceModel, X=None, x_const: Optional[float] = None,
                mode: int = MODE_LAYERED, out=None):
        """scores[num_nodes, out_dim] (float32) = model.outputs for every node of the batch."""
        return self._forward(b, self.supports(b), model, X, x_const, mode, out)

    def _forward(self, b, lap, model, X, x_const, mode, out):
        t = self.torch
        if x_const is None:
            x_const = float(np.float32(1.0 / model.in_dim))  # row-normalised all-ones features
        if out is None:
            out = t.empty((b.host.num_nodes, model.out_dim), dtype=t.float32, device=self.device)
        if model.num_supports == 3:  # [I, L, L.L]: layer by layer through the poly entry
            if mode != MODE_LAYERED:
                raise _lib.DgcnError("max_degree=2 models run layer by layer (mode=MODE_LAYERED)")
            lap2 = self.supports2(b)
            need = int(self.lib.dgcn_gcn_forward_workspace(C.byref(b.c), C.byref(model.c), 0))
            ws = self._workspace(need)
            sups = (C.POINTER(_lib.DgcnCsr) * 2)(C.pointer(lap["c"]), C.pointer(lap2["c"]))
            _lib.check(self.lib.dgcn_gcn_forward_poly_batch(C.byref(b.c), sups, C.byref(model.c),
                                                            X.data_ptr() if X is not None else None, x_const,
                                                            out.data_ptr(), ws.data_ptr(), int(ws.numel()), self._stream()),
                       "dgcn_gcn_forward_poly_batch")
            return out
        need = int(self.lib.dgcn_gcn_forward_workspace(C.byref(b.c), C.byref(model.c), mode))
        if need == 0:
            _lib.check(-1, "dgcn_gcn_forward_workspace")
        ws = self._workspace(need)
        _lib.check(self.lib.dgcn_gcn_forward_batch(C.byref(b.c), C.byref(lap["c"]), C.byref(model.c),
                                                   X.data_ptr() if X is not None else None, x_const, out.data_ptr(),
                                                   ws.data_ptr(), int(ws.numel()), mode, self._stream()),
                   "dgcn_gcn_forward_batch")
        return out

    def model_bank(self, models, precision: str = "float32") -> ModelBank:
        """Checkpoints of one architecture ([I, L] supports) as a bank.  ``models``: a list of what ``DeviceModel`` takes (or of
        objects with such ``.layers``, e.g. ``gcn.models.GCN_DQN``).  ``precision="int8"``: the products of the hidden layers run in 8-bit integers
        with scales per vertex and output column; the first and the last layer stay in float32 (as do all aggregations).

        A bank is for many models in one batch: its time does not depend on their number, while ``solve_fused`` on each model's part of the
        batch is a launch per model and faster up to three or four of them (500 graphs of 200 vertices: 20 layers 32 wide 604 us against
        199 with one model, 538 with four, 804 with six; 6 layers 204 against 80 with one, 168 with three, 226 with four).  8 bits pay from 64
        columns on (six layers, 64 wide: 304 us against 339; 128 wide: 570 against 794) and cost time below (32 wide: 185 against 173)."""
        t = self.torch
        models = list(models)
        if any(getattr(m, "has_head", False) for m in models):
            raise _lib.DgcnError("a bank takes models whose output is their last layer (no is_dual / skip head)")
        models = [getattr(m, "layers", m) for m in models]
        if not models or not models[0]:
            raise ValueError("a bank needs at least one model with at least one layer")
        if precision not in ("float32", "int8"):
            raise ValueError("precision %r: float32 or int8" % (precision,))
        shape = lambda m: [([np.shape(w) for w in lyr["weights"]], lyr.get("bias") is not None, ACT_CODES[lyr.get("act")]) for lyr in m]
        for k, m in enumerate(models):
            if shape(m) != shape(models[0]):
                raise ValueError("model %d differs from model 0 in layers, supports, widths, bias or activation" % k)
        layers = []
        for l, proto in enumerate(models[0]):
            if len(proto["weights"]) != 2:
                raise _lib.DgcnError("a bank takes [I, L] models (max_degree=1); layer %d has %d supports" % (l, len(proto["weights"])))
            fin, fout = np.shape(proto["weights"][0])
            if l and fin != layers[-1]["out"]:
                raise ValueError("layer %d takes %d features, layer %d gives %d" % (l, fin, l - 1, layers[-1]["out"]))
            W = np.stack([np.concatenate([np.asarray(w, dtype=np.float32) for w in m[l]["weights"]], axis=1).T for m in models])
            W = t.from_numpy(np.ascontiguousarray(W)).to(self.device)
            bias = None
            if proto.get("bias") is not None:
                bias = np.stack([np.concatenate([np.asarray(m[l]["bias"], dtype=np.float32).ravel(), np.zeros(fout, np.float32)]) for m in models])
                bias = t.from_numpy(bias).to(self.device)
            q = scale = None
            if precision == "int8" and 0 < l < len(models[0]) - 1:
                q, scale = self.quantize_rows(W.reshape(-1, fin))
                q, scale, W = q.reshape(W.shape), scale.reshape(W.shape[:2]), None
            layers.append({"weights": W, "bias": bias, "act": proto.get("act"), "in": int(fin), "out": int(fout), "q": q, "scale": scale})
        return ModelBank(layers, len(models), precision)

    def forward_bank(self, b: DeviceBatch, bank: ModelBank, model_of_graph, X=None, x_const: Optional[float] = None, status=None):
        """scores[num_nodes, out_dim] of a batch whose graph g belongs to model ``model_of_graph[g]`` (int32 on the device), layer by
        layer, one product and one aggregation launch each for the whole batch.  A float32 bank without biases returns the bits of
        ``forward`` with each graph's own model (biases are added before the neighbours' sum here and behind it there); an 8-bit bank is
        an approximation whose error is the quantisation's.  ``status``: as in ``transform_grouped``; the faults of the batch's
        adjacency (``supports``) are reported by every call - with ``status`` by a small launch more (about 4 us where the host is the bound),
        until ``supports(b)`` or a call without ``status`` has read that there are none."""
        scores, word = self._forward_bank(b, bank, model_of_graph, X, x_const, status)
        if status is None and b.host.num_nodes:
            self.check_status(word)
            b.lap["checked"] = True
        return scores

    def _forward_bank(self, b, bank, model_of_graph, X, x_const, status):
        """-> (scores, status word: the caller's, or one of this call with the faults of the batch's supports)."""
        t = self.torch
        B, n = b.host.num_graphs, b.host.num_nodes
        _array(model_of_graph, "model_of_graph", t.int32, (B,))
        if X is not None:
            _matrix(X, "X", (t.float32,), cols=bank.in_dim, rows=n)
        self._here(model_of_graph, X)
        if n == 0:
            return (t.empty((0, bank.out_dim), dtype=t.float32, device=self.device),
                    t.zeros(1, dtype=t.int32, device=self.device) if status is None else status)
        if x_const is None:
            x_const = float(np.float32(1.0 / bank.in_dim))
        if b.lap is None and t.cuda.is_current_stream_capturing():
            raise _lib.DgcnError("the batch's supports are made once and kept: call supports(b) before the capture")
        with t.cuda.device(self._index()):
            if status is None:
                status, lap = self._call_status(b), b.lap
            else:
                lap = self.supports(b, status=status)
            H = X
            for l, lyr in enumerate(bank.layers):
                out = lyr["out"]
                if lyr["q"] is not None:
                    q, s = self.quantize_rows(H)
                    Z = self.transform_grouped_int8(q, s, lyr["q"], lyr["scale"], b.graph_ptr, model_of_group=model_of_graph,
                                                    bias=lyr["bias"], status=status)
                else:
                    Z = self.transform_grouped(H, lyr["weights"], b.graph_ptr, model_of_group=model_of_graph, bias=lyr["bias"], rows=n,
                                               h_const=x_const, precise=l == 1, status=status)
                H = self.spmm(lap, Z[:, out:], out, ldz=2 * out, graph_ptr=b.graph_ptr, num_graphs=B, max_nodes=b.host.max_nodes, Y0=Z,
                              ldy0=2 * out, act=lyr["act"], precise=l == 0)
        return H, status

    def head_dual(self, b: DeviceBatch, act):
        """GCN2_DQN(is_dual=True) output head (gcn/models.py:651-653): [num_nodes, D] -> [num_nodes, D - 1]."""
        t = self.torch
        D = int(act.shape[1])
        out = t.empty((b.host.num_nodes, D - 1), dtype=t.float32, device=self.device)
        _lib.check(self.lib.dgcn_head_dual_batch(act.data_ptr(), D, b.graph_ptr.data_ptr(), b.host.num_graphs, out.data_ptr(),
                                                 self._stream()), "dgcn_head_dual_batch")
        return out

    def head_skip(self, act, kernel, bias, X=None, x_const: float = 1.0, in_dim: int = 1):
        """GCN_DQN(skip=True) output head (gcn/models.py:505-521): dense(concat([X, act])) -> [num_nodes, D]."""
        t = self.torch
        out = t.empty_like(act)
        _lib.check(self.lib.dgcn_head_skip_batch(X.data_ptr() if X is not None else None, x_const, in_dim, act.data_ptr(),
                                                 int(act.shape[1]), kernel.data_ptr(), bias.data_ptr() if bias is not None else None,
                                                 int(act.shape[0]), out.data_ptr(), self._stream()), "dgcn_head_skip_batch")
        return out

    def argmax(self, b: DeviceBatch, scores):
        t = self.torch
        out = t.empty(b.host.num_graphs, dtype=t.int32, device=self.device)
        _lib.check(self.lib.dgcn_argmax_batch(scores.data_ptr(), int(scores.shape[-1]) if scores.dim() > 1 else 1,
                                              b.graph_ptr.data_ptr(), b.host.num_graphs, out.data_ptr(),
                                              self._stream()), "dgcn_argmax_batch")
        return out

    # ------------------------------------------------------------------ A7-A9
    def lgs(self, b: DeviceBatch, prio=None, scores=None, weights=None, max_rounds: int = 0, want_stats=False,
            want_overhead=False, sum_weights=None, want_totals=True, status=None):
        """Local greedy search over the batch.  Returns a dict of device tensors."""
        n, B = b.host.num_nodes, b.host.num_graphs
        own = status is None
        pk = self._packed([("totals", max(B, 1) if want_totals else 0, "float64"),
                           ("stats", 2 * max(B, 1) if want_stats or want_overhead else 0, "int64"),
                           ("rounds", max(B, 1), "int32"), ("overhead", max(n, 1) if want_overhead else 0, "int32"),
                           ("status", 1 if own else 0, "int32"), ("state", max(n, 1), "uint8")])
        state, rounds, totals, overhead = pk["state"], pk["rounds"], pk["totals"], pk["overhead"]
        stats = pk["stats"].reshape(-1, 2) if pk["stats"] is not None else None
        if own:
            status = pk["status"]
        p = lambda x: x.data_ptr() if x is not None else None
        _lib.check(self.lib.dgcn_lgs_batch(C.byref(b.c), p(prio), p(scores), p(weights), int(max_rounds), p(state),
                                           p(rounds), p(stats), p(overhead), p(sum_weights), p(totals), p(status),
                                           self._stream()), "dgcn_lgs_batch")
        return {"state": state[:n], "rounds": rounds[:B], "stats": stats, "overhead": overhead,
                "totals": totals, "status": status, "flat": pk["flat"], "layout": pk["layout"]}

    def margin_risk(self, b: DeviceBatch, state, delta: float, prio=None, scores=None, weights=None):
        """per graph, the number of excluded vertices whose exclusion a score error of ``delta`` could
        overturn (``dgcn_margin_risk_batch``); 0 proves the graph's set is the same for every score vector within
        ``delta`` of this one.  -> int32 device tensor [num_graphs]."""
        t = self.torch
        out = t.zeros(max(b.host.num_graphs, 1), dtype=t.int32, device=self.device)
        p = lambda x: x.data_ptr() if x is not None else None
        _lib.check(self.lib.dgcn_margin_risk_batch(C.byref(b.c), p(prio), p(scores), p(weights), state.data_ptr(),
                                                   float(delta), out.data_ptr(), self._stream()), "dgcn_margin_risk_batch")
        return out[:b.host.num_graphs]

    def lgs_masked(self, b: DeviceBatch, prio, init_state, num_instances: int, sum_weights=None, max_rounds: int = 0,
                   prio_stride: int = 0):
        """Greedy search on ``num_instances`` residuals of the same batch (``dgcn_lgs_masked_batch``).
        ``init_state`` is uint8 ``[num_instances, num_nodes]`` (non-zero = vertex taken out)."""
        t = self.torch
        n, B = b.host.num_nodes, b.host.num_graphs
        state = t.empty((num_instances, max(n, 1)), dtype=t.uint8, device=self.device)
        rounds = t.empty((num_instances, max(B, 1)), dtype=t.int32, device=self.device)
        totals = t.empty((num_instances, max(B, 1)), dtype=t.float64, device=self.device)
        status = t.zeros(1, dtype=t.int32, device=self.device)
        _lib.check(self.lib.dgcn_lgs_masked_batch(C.byref(b.c), prio.data_ptr(), int(prio_stride), init_state.data_ptr(),
                                                  int(num_instances), int(max_rounds), state.data_ptr(), rounds.data_ptr(),
                                                  sum_weights.data_ptr() if sum_weights is not None else None,
                                                  totals.data_ptr(), status.data_ptr(), self._stream()),
                   "dgcn_lgs_masked_batch")
        return {"state": state[:, :n], "rounds": rounds[:, :B], "totals": totals[:, :B], "status": status}

    # ------------------------------------------------------------------ A10 (batched)
    def _empty_solution(self, b: DeviceBatch, status):
        """Nothing but empty graphs: rounds 0, totals 0 (heuristics.py loops do not run)."""
        t = self.torch
        B = b.host.num_graphs
        return {"state": t.empty(0, dtype=t.uint8, device=self.device),
                "rounds": t.zeros(B, dtype=t.int32, device=self.device),
                "totals": t.zeros(B, dtype=t.float64, device=self.device), "status": status,
                "scores": t.empty((0, 1), dtype=t.float32, device=self.device), "stats": None, "overhead": None}

    def solve(self, b: DeviceBatch, model: DeviceModel, predict: str = "mwis", mode: int = MODE_LAYERED, X=None,
              x_const=None):
        """GCN forward -> priority -> local greedy for every graph of the batch
        (mwis_gdpg_call.py:200-235, batched).  ``b.weights`` must be set."""
        if b.weights is None:
            raise ValueError("batch has no vertex weights")
        if model.out_dim != 1:
            raise _lib.DgcnError("solve() needs a model with one output per node (diver_num=1)")
        if b.host.num_nodes == 0:
            return self._empty_solution(b, self.torch.zeros(1, dtype=self.torch.int32, device=self.device))
        if mode == MODE_FUSED:
            return self.solve_fused(b, model, predict=predict, X=X, x_const=x_const)
        status = self._call_status(b)  # no host sync on the path: faults surface through res["status"]
        scores = self._forward(b, b.lap, model, X, x_const, mode, None)
        res = self.lgs(b, scores=scores, weights=b.weights if predict == "mwis" else None, sum_weights=b.weights,
                       status=status)
        res["scores"] = scores
        return res

    def solve_bank(self, b: DeviceBatch, bank: ModelBank, model_of_graph, predict: str = "mwis", X=None, x_const=None):
        """``solve`` for a batch whose graphs belong to different models: ``forward_bank`` -> priority -> local greedy.  Faults surface
        through ``res["status"]``."""
        if b.weights is None:
            raise ValueError("batch has no vertex weights")
        if bank.out_dim != 1:
            raise _lib.DgcnError("solve_bank() needs models with one output per node (diver_num=1)")
        scores, status = self._forward_bank(b, bank, model_of_graph, X, x_const, None)
        if b.host.num_nodes == 0:
            return self._empty_solution(b, status)
        res = self.lgs(b, scores=scores, weights=b.weights if predict == "mwis" else None, sum_weights=b.weights, status=status)
        res["scores"] = scores
        return res

    def solve_supported(self, b: DeviceBatch, model: DeviceModel) -> bool:
        """Does the per-graph fused kernel (one workgroup, one graph, everything in LDS) take this batch?"""
        return bool(self.lib.dgcn_solve_supported(C.byref(b.c), C.byref(model.c)))

    def solve_path(self, b: DeviceBatch, model: DeviceModel) -> int:
        """What ``solve_fused`` / ``solve_residual`` (``dgcn_solve_batch`` / ``dgcn_solve_residual_batch``) will run:
        1 = the fused kernels, 2 = the any-size device path (``csrc/general.hip``: graphs beyond 512 vertices or one
        CU's LDS, layer stacks wider than 32), 0 = neither."""
        return int(self.lib.dgcn_solve_path(C.byref(b.c), C.byref(model.c)))

    def solve_buffers(self, b: DeviceBatch, want_scores: bool = True, cap_nodes: int = 0, cap_graphs: int = 0):
        """Output buffers of ``solve_fused`` for a batch, for callers that re-use them across calls
        (a steady-state serving loop should not pay five allocations per batch).  All of them are views
        into ONE byte tensor, so everything comes back with a single device-to-host copy
        (``fetch_solve_buffers``) - or goes out in a single collective (``out["flat"]`` is what bench.py
        all-gathers: membership + totals + rounds + status of a rank in one buffer).  ``cap_nodes`` /
        ``cap_graphs``: lay the buffer out for that many vertices / graphs (every rank of a sharded batch
        uses the largest shard's sizes, so all ranks' buffers have one layout)."""
        n, B = max(b.host.num_nodes, cap_nodes, 1), max(b.host.num_graphs, cap_graphs, 1)
        out = self._packed(solve_buffer_specs(n, B, want_scores))
        if want_scores:
            out["scores"] = out["scores"].reshape(n, 1)
        return out

    @classmethod
    def fetch_solve_buffers(cls, out, num_nodes: int, num_graphs: int):
        """-> dict of NumPy arrays (state, totals, rounds, scores or None, status as int)."""
        h = cls.fetch_packed(out)
        return {"state": h["state"][:num_nodes], "totals": h["totals"][:num_graphs], "rounds": h["rounds"][:num_graphs],
                "scores": h["scores"][:num_nodes].reshape(-1, 1) if "scores" in h else None,
                "status": int(h["status"][0])}

    def solve_fused(self, b: DeviceBatch, model: DeviceModel, predict: str = "mwis", X=None, x_const=None,
                    want_scores: bool = True, out=None):
        """The whole path in one launch (dgcn_solve_batch): adjacency + weights in, membership out.
        ``out`` = buffers from ``solve_buffers`` to re-use (its status word accumulates faults)."""
        n, B = b.host.num_nodes, b.host.num_graphs
        if x_const is None:
            x_const = float(np.float32(1.0 / model.in_dim))
        tab = self._dinv(b.host.max_degree)
        if out is None:
            out = self.solve_buffers(b, want_scores)
        scores, state, rounds, totals, status = out["scores"], out["state"], out["rounds"], out["totals"], out["status"]
        p = lambda x: x.data_ptr() if x is not None else None
        need = int(self.lib.dgcn_solve_workspace(C.byref(b.c), C.byref(model.c)))
        ws = self._workspace(need)
        _lib.check(self.lib.dgcn_solve_batch(C.byref(b.c), C.byref(model.c), tab.data_ptr(), int(tab.numel()), p(X),
                                             x_const, p(b.weights), 1 if predict == "mwis" else 0, p(scores),
                                             p(state), p(rounds), p(totals), p(status), ws.data_ptr(), need,
                                             self._stream()),
                   "dgcn_solve_batch")
        return {"state": state[:n], "rounds": rounds[:B], "totals": totals[:B], "status": status,
                "scores": None if scores is None else scores[:n], "stats": None, "overhead": None}

    GREEDY_ROUNDS, GREEDY_CENTRAL, GREEDY_ROLLOUT = 0, 1, 2
    SCORES_GIVEN, COMPLETE_BY_PRIORITY, FINISH_SMALL = 1, 2, 4  # DGCN_RESIDUAL_* option bits

    def solve_residual(self, b: DeviceBatch, model: DeviceModel, state, predict: str = "mwis", greedy: int = 0,
                       max_rounds: int = 0, beam: int = 16, X=None, x_const=None, weight_features: bool = False,
                       want_scores: bool = False, max_steps: Optional[int] = None, out=None, options: int = 0,
                       scores=None, finish_small: Optional[bool] = None):
        """Iterative solvers on the device (dgcn_solve_residual_batch): repeat one launch per step on the
        residual graphs until no graph makes progress.  ``state`` (uint8 [num_nodes], 0 = undecided) is
        updated in place.  greedy = GREEDY_ROUNDS with max_rounds=1 is solve_mwis_dit, GREEDY_CENTRAL is
        solve_mwis_cit, GREEDY_ROLLOUT is solve_mwis_rollout (mwis_gdpg_call.py:278-318, 343-384, 596-659)
        for every graph of the batch at once.  -> {"state", "steps", "status", "scores" (last step)}
        ``finish_small`` (default: on for a search run to its end, off when ``max_steps`` asks for single steps): a graph
        with at most 64 undecided vertices runs the rest of its search inside the call that finds it so
        (DGCN_RESIDUAL_FINISH_SMALL, csrc/tail.hip); same final states, fewer calls - ``steps`` counts calls."""
        t = self.torch
        n, B = b.host.num_nodes, b.host.num_graphs
        if x_const is None:
            x_const = float(np.float32(1.0 / model.in_dim))
        tab = self._dinv(b.host.max_degree)
        if out is None:
            out = self.solve_buffers(b, want_scores)
        if options & self.SCORES_GIVEN:
            if scores is None:
                raise ValueError("options & SCORES_GIVEN needs scores")
            out = dict(out, scores=scores)
        if finish_small is None:
            finish_small = max_steps is None
        p = lambda x: x.data_ptr() if x is not None else None
        need = int(self.lib.dgcn_solve_workspace(C.byref(b.c), C.byref(model.c)))
        ws = self._workspace(need)
        steps = 0
        limit = max_steps if max_steps is not None else max(b.host.max_nodes, 1) + 1
        # Steps are launched a few at a time, each with its own progress word, and the words are read back together: a
        # step that decides nothing leaves the state as it is, so every later step of the group decides nothing either
        # (and costs next to nothing: a graph with nothing left returns at once) - one host round trip per group, not per step.
        group = 4
        issued = 0
        done = n == 0
        # (the status word is sticky - kernels OR into it, nobody clears it: only bits set DURING this search end it, a fault
        # an earlier call left in a re-used `out` is the caller's to read, not a reason to cut this search short)
        status_at_entry = out["status"].reshape(-1)[:1].to(t.int32).clone()
        while not done and steps < limit:
            k = min(group, limit - steps)
            progress = t.zeros(k, dtype=t.int32, device=self.device)
            for i in range(k):
                # (the tail's launch leaves at once while a graph of the batch is still large: asked for with every second
                # call, it costs a search ~3 us per step and starts at most one step late)
                opts = options | (self.FINISH_SMALL if finish_small and ((issued + i) & 1) else 0)
                _lib.check(self.lib.dgcn_solve_residual_batch(
                    C.byref(b.c), C.byref(model.c), tab.data_ptr(), int(tab.numel()), p(X), x_const,
                    1 if weight_features else 0, p(b.weights), 1 if predict == "mwis" else 0, int(greedy),
                    int(max_rounds), int(beam), int(opts), p(out["scores"]), state.data_ptr(), p(out["rounds"]), p(out["totals"]),
                    progress.data_ptr() + 4 * i, out["status"].data_ptr(), ws.data_ptr(), need, self._stream()),
                    "dgcn_solve_residual_batch")
            issued += k
            if max_steps == 1:  # a caller that asks for exactly one step does not need to know whether it decided anything
                steps = 1
                break
            # (the status word rides along: a fault such as a NaN priority leaves its graph undecided - "active" - for ever,
            # and the any-size path counts active graphs as progress; the caller's check_status reports it)
            words = t.cat([progress, out["status"].reshape(-1)[:1].to(t.int32), status_at_entry]).cpu().tolist()
            for v in words[:k]:
                if v == 0:
                    done = True
                    break
                steps += 1
            fresh = words[k] & ~words[k + 1]
            if fresh == 16:
                # a placement fault of the several-workgroups-per-graph launch (automatic for searches on small batches): the
                # step left the searches it touched as they were (fused.hip) - switch the variant off, clear the bit, go on
                self.lib.dgcn_set_cluster(0)
                out["status"].bitwise_and_(~16)
                done = False
            elif fresh:
                done = True
            group = min(2 * group, 32)  # (a search of ~100 steps: 6 read-backs instead of 14; at most 31 empty launches at its end)
        return {"state": state, "steps": steps, "status": out["status"],
                "scores": None if out["scores"] is None else out["scores"][:n]}

    # ------------------------------------------------------------------ timing hooks (bench.py)
    def timing(self, on: bool):
        """on=True clears earlier records and starts recording; on=False stops (records stay readable)."""
        if on:
            self.lib.dgcn_timing_reset()
        # (DGCN_TIMING_EVERY=N: an event pair round every N-th launch only - an A/B switch for what the instrumentation costs;
        # anything below 1 means 1: "on" never silently turns the recording off)
        self.lib.dgcn_timing_enable(max(1, int(os.environ.get("DGCN_TIMING_EVERY", "1"))) if on else 0)

    def timing_read(self, family: str):
        """(milliseconds, launches) of a kernel family since timing(True).  With every N-th launch sampled both are scaled by N
        (estimates of the whole region: the average per launch is unchanged, per-step figures stay per step)."""
        ms = C.c_double(0.0)
        n = C.c_int64(0)
        _lib.check(self.lib.dgcn_timing_read(family.encode(), C.byref(ms), C.byref(n)), "dgcn_timing_read")
        every = max(1, int(self.lib.dgcn_timing_sampling()))
        return ms.value * every, n.value * every
