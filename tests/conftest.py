import os
import sys

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)
GOLDEN = os.path.join(ROOT, "tests", "golden")


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu on the GPU box)")


def pytest_collection_modifyitems(config, items):
    """The tests that run the reference itself need its files: an empty folder in its place holds none."""
    ref = os.environ.get("DGCN_REFERENCE", "/root/reference")
    if not os.path.isfile(os.path.join(ref, "heuristics.py")):
        for item in items:
            if item.name in ("test_reference_import_agrees_when_available", "test_reference_execution_is_reproducible_when_available"):
                item.add_marker(pytest.mark.skip(reason="reference tree not present"))


class Golden:
    """Fixture data generated by oracle/make_golden.py from the imported reference."""

    def __init__(self):
        self.graphs = np.load(os.path.join(GOLDEN, "graphs.npz"))
        self.supports = np.load(os.path.join(GOLDEN, "supports.npz"))
        self.lgs = np.load(os.path.join(GOLDEN, "lgs.npz"))
        self.models = np.load(os.path.join(GOLDEN, "models.npz"))
        self.scores = np.load(os.path.join(GOLDEN, "scores.npz"))
        self.names = [str(x) for x in self.graphs["names"]]
        self.model_names = [str(x) for x in self.models["names"]]
        self.num_graphs = len(self.names)

    def csr(self, i):
        k = "g%02d" % i
        return self.graphs[k + "_indptr"], self.graphs[k + "_indices"], self.graphs[k + "_weights"]

    def scipy(self, i):
        import scipy.sparse as sp
        p, c, w = self.csr(i)
        return sp.csr_matrix((np.ones(c.size), c, p), shape=(w.size, w.size))

    def host_batch(self, ids=None):
        from distgcn_amd.batch import HostBatch
        ids = range(self.num_graphs) if ids is None else ids
        ps, cs, ws = [], [], []
        for i in ids:
            p, c, w = self.csr(i)
            ps.append(p.astype(np.int64))
            cs.append(c.astype(np.int64))
            ws.append(w)
        return HostBatch.from_csr_lists(ps, cs, ws)

    def params(self, model_name):
        pre = model_name + "|"
        return {k[len(pre):]: self.models[k] for k in self.models.files if k.startswith(pre)}

    def layers(self, model_name):
        from oracle import ref_numpy as orc
        return orc.gcn_layer_specs(self.params(model_name))


class AllModels:
    """tests/golden/all_models.npz (oracle/make_golden_models.py): every shipped checkpoint (44 cheb1 + 2 cheb2)."""

    def __init__(self):
        self.z = np.load(os.path.join(GOLDEN, "all_models.npz"))
        self.names = [str(n) for n in self.z["names"]]
        self.graph_ids = [int(g) for g in self.z["graphs"]]

    def params(self, name):
        pre = name + "|"
        return {k[len(pre):]: self.z[k] for k in self.z.files
                if k.startswith(pre) and not k.endswith("|meta")}

    def layers(self, name):
        from distgcn_amd.gcn.models import layers_from_params
        return layers_from_params(self.params(name))

    def meta(self, name):
        f, c, l, md = (int(v) for v in self.z[name + "|meta"])
        return {"feature_size": f, "hidden": c, "num_layer": l, "max_degree": md,
                "predict": "mis" if name.endswith("_mis_dqn") else "mwis"}

    def expect(self, gi, name, what):
        return self.z["g%02d|%s|%s" % (gi, name, what)]


class Dataset100:
    """tests/golden/dataset100.npz (oracle/make_golden_dataset.py): 50 ER + 50 BA graphs of the reference's test2
    folders with the known answers stored in / derived from the reference."""

    def __init__(self):
        self.z = np.load(os.path.join(GOLDEN, "dataset100.npz"))
        self.names = [str(n) for n in self.z["names"]]
        self.n = len(self.names)

    def csr(self, i):
        return self.z["indptr_%d" % i], self.z["indices_%d" % i].astype(np.int32), self.z["weights_%d" % i]

    def host_batch(self, weights=True):
        from distgcn_amd.batch import HostBatch
        parts = [self.csr(i) for i in range(self.n)]
        return HostBatch.from_csr_lists([p[0] for p in parts], [p[1] for p in parts],
                                        [p[2] for p in parts] if weights else None)


TOL = 1e-5  # north star: node scores within 1e-5


def check_scores(got, f32, f64, what=None, strict=False):
    """The score bar, in one place.  (1) Within 1e-5 of the exact value (the float64 evaluation of the reference's
    formula).  ``strict`` (the BASELINE configurations at full size): always.  Otherwise (any shipped model on any
    fixture graph, out-of-distribution pairs included: a BA-trained 20-layer model on an ER p = 0.02 forest): or at
    least no further from it than the float32 restatement is - float32 hidden layers cannot promise more than float32.
    (2) Within 1e-5 of the float32 restatement too - a SECOND float32 evaluation with rounding errors of its own (at
    l = 20 up to 1.4e-5 from the exact value on hub-heavy graphs) - unless on that graph the restatement is the one
    further from the exact value.  Errors are measured in units of max(1, |score|): 1e-5 is absolute for the
    mwis models (|score| <= 2) and relative for the one shipped model whose scores reach 21 (F = 32, predict = mis:
    float32 spacing 1.9e-6 there).  Returns the three maxima (|got - f32|, |got - f64|, |f32 - f64|) in those units."""
    got, f32, f64 = np.asarray(got).ravel(), np.asarray(f32).ravel(), np.asarray(f64).ravel()
    unit = np.maximum(1.0, np.abs(f64))
    e64 = float((np.abs(got - f64) / unit).max())
    e32 = float((np.abs(got.astype(np.float64) - f32) / unit).max())
    e3264 = float((np.abs(f32.astype(np.float64) - f64) / unit).max())
    assert e64 <= (TOL if strict else max(TOL, e3264)), (what, "vs float64", e64, e3264)
    assert e32 <= TOL or e64 < e3264, (what, "vs float32 restatement", e32, e64, e3264)
    return e32, e64, e3264


@pytest.fixture(scope="session")
def golden():
    return Golden()


@pytest.fixture(scope="session")
def dataset100():
    return Dataset100()


@pytest.fixture(scope="session")
def all_models():
    return AllModels()


@pytest.fixture(scope="session")
def engine():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from distgcn_amd.engine import Engine
    return Engine("cuda:0")


@pytest.fixture(autouse=True)
def _options_as_the_process_started(request):
    """Every GPU test ends with the library's option table (dgcn_set_option) as the process started - a test that flips a path
    switch and fails half-way must not send the rest of the suite down that path."""
    if "gpu" not in request.keywords:
        yield
        return
    from distgcn_amd import _lib
    before = {k: _lib.get_option(k) for k in _lib.option_defaults()}
    yield
    for k, v in before.items():
        if _lib.get_option(k) != v:
            _lib.set_option(k, v)


@pytest.fixture
def cluster_switch():
    """Sets the library's several-workgroups-per-graph switch (dgcn_set_cluster: -1 automatic, 0 off, K forced) for the
    duration of a test and puts back whatever the process started with (e.g. a suite run with DGCN_OPTIONS="fused_cluster=8")."""
    from distgcn_amd import _lib
    lib = _lib.load()
    initial = int(lib.dgcn_get_cluster())

    def set_to(value):
        lib.dgcn_set_cluster(-1 if value is None else int(value))
    yield set_to
    lib.dgcn_set_cluster(initial)


def pytest_sessionfinish(session, exitstatus):
    """Leave the process in a defined state before the interpreter starts tearing it down: every host-solver object that is
    still open (the process-wide one-slot instances behind heuristics.* / solve_mwis are never closed by their users) is closed
    here - streams drained, pinned and device buffers released while the HIP runtime is certainly still alive - and the device
    is idle."""
    try:
        import torch
        if not torch.cuda.is_available():
            return
        from distgcn_amd import serving
        serving._close_all()
        torch.cuda.synchronize()
    except Exception:
        pass
