"""GPU: batches of several models when something is wrong with the batch - what is reported, how often, and what the launches behind the
report may touch."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _graphs(sizes, seed):
    import scipy.sparse as sp
    rng = np.random.default_rng(seed)
    adjs = []
    for n in sizes:
        a = np.triu(rng.random((n, n)) < min(1.0, 12.0 / max(n, 1)), 1)
        adjs.append(sp.csr_matrix((a + a.T).astype(float)))
    return adjs, [rng.random(n) for n in sizes]


def _batch_with_columns(sizes, seed, where):
    """A batch whose entries ``where`` = {(graph, entry of the graph): column id of the batch} point elsewhere."""
    from distgcn_amd.batch import HostBatch
    good = HostBatch.from_scipy(*_graphs(sizes, seed))
    col = good.col_idx.copy()
    for (g, e), c in where.items():
        col[good.row_ptr[good.graph_ptr[g]] + e] = c
    return good, HostBatch(good.graph_ptr, good.row_ptr, col, good.weights)


FAR = {(1, 0): 2 ** 31 - 1, (1, 5): -1, (1, 9): -(2 ** 31), (3, 2): 0, (3, 40): 10 ** 6}


@pytest.mark.parametrize("sizes", [[30, 50, 20, 70], [200, 900, 100, 300]])
def test_columns_outside_their_graph_are_reported_and_never_followed(engine, sizes):
    import torch
    from distgcn_amd import datagen
    from distgcn_amd._lib import DgcnError
    from distgcn_amd.engine import DeviceModel
    good, bad = _batch_with_columns(sizes, 1, FAR)
    ok = [(lo, hi) for g, (lo, hi) in enumerate(good.graph_slices()) if g not in (1, 3)]
    models = [datagen.random_model(3, 16, seed=s) for s in (1, 2)]
    mog = torch.tensor([0, 1, 1, 0], dtype=torch.int32, device="cuda:0")
    bank, dm = engine.model_bank(models), DeviceModel(models[0], "cuda:0")

    status = torch.zeros(1, dtype=torch.int32, device="cuda:0")
    lap = engine.supports(engine.upload(bad), status=status)
    assert int(status) == 8
    col, val, row = (lap[k].cpu().numpy() for k in ("col_idx", "values", "row_ptr"))
    own = np.repeat(np.arange(bad.num_nodes), np.diff(row))
    graph = np.repeat(np.arange(4), sizes)
    assert np.array_equal(graph[col], graph[own])
    for (g, e), c in FAR.items():
        at = good.row_ptr[good.graph_ptr[g]] + e
        at += int(np.searchsorted(good.row_ptr, at, side="right"))  # a diagonal entry in front of every row
        assert col[at] == own[at] and val[at] == 0

    with pytest.raises(DgcnError, match="column index"):
        engine.forward_bank(engine.upload(bad), bank, mog)
    clean = engine.solve_bank(engine.upload(good), bank, mog)
    res = engine.solve_bank(engine.upload(bad), bank, mog)
    assert int(clean["status"]) == 0 and int(res["status"]) & 8
    one = engine.solve(engine.upload(bad), dm)
    assert int(one["status"]) & 8
    one_clean = engine.solve(engine.upload(good), dm)
    for lo, hi in ok:  # the other graphs of the batch are what they are without it
        for a, b in ((res, clean), (one, one_clean)):
            assert torch.equal(a["scores"][lo:hi], b["scores"][lo:hi]) and torch.equal(a["state"][lo:hi], b["state"][lo:hi])


@pytest.mark.parametrize("kw", [{}, {"want_stats": True}, {"max_rounds": 1}])
@pytest.mark.parametrize("sizes,degree", [([30, 50, 20, 70], 12), ([20, 2000, 30, 100], 80)])
def test_greedy_search_stays_inside_its_graph(engine, sizes, degree, kw):
    """Columns outside the graph, with the columns in LDS and - 2 000 vertices of 80 neighbours - in global memory."""
    import torch
    import scipy.sparse as sp
    from distgcn_amd.batch import HostBatch
    rng = np.random.default_rng(4)
    adjs = []
    for n in sizes:
        a = np.triu(rng.random((n, n)) < min(1.0, degree / n), 1)
        adjs.append(sp.csr_matrix((a + a.T).astype(float)))
    good = HostBatch.from_scipy(adjs, [rng.random(n) for n in sizes])
    col = good.col_idx.copy()
    for (g, e), c in FAR.items():
        col[good.row_ptr[good.graph_ptr[g]] + e] = c
    bad = HostBatch(good.graph_ptr, good.row_ptr, col, good.weights)
    prio = torch.from_numpy(rng.random(good.num_nodes)).cuda()
    a, b = engine.lgs(engine.upload(good), prio=prio, **kw), engine.lgs(engine.upload(bad), prio=prio, **kw)
    for g, (lo, hi) in enumerate(good.graph_slices()):
        state = b["state"][lo:hi]
        assert int(state.max()) <= 2 and (kw.get("max_rounds") or int(state.min()) >= 1)
        if g in (0, 2):
            assert torch.equal(state, a["state"][lo:hi]) and int(a["rounds"][g]) == int(b["rounds"][g])


def test_margin_risk_stays_inside_its_graph(engine):
    """A column outside the graph is nobody's member neighbour."""
    import torch
    good, bad = _batch_with_columns([30, 50, 20, 70], 1, FAR)
    prio = torch.from_numpy(np.random.default_rng(5).random(good.num_nodes)).cuda()
    a, b = engine.upload(good), engine.upload(bad)
    state = engine.lgs(a, prio=prio)["state"]
    want, got = (engine.margin_risk(x, state, 1e-3, prio=prio).cpu().numpy() for x in (a, b))
    assert want[0] == got[0] and want[2] == got[2]
    # by the definition: an excluded vertex is safe iff a member neighbour is ahead by more than twice delta
    st, p = state.cpu().numpy(), prio.cpu().numpy()
    for g, (lo, hi) in enumerate(bad.graph_slices()):
        risky = 0
        for v in range(lo, hi):
            near = bad.col_idx[bad.row_ptr[v]:bad.row_ptr[v + 1]]
            near = near[(near >= lo) & (near < hi)]
            risky += st[v] == 2 and not any(st[u] == 1 and p[u] - p[v] > 2e-3 for u in near)
        assert got[g] == risky, g


def _self_loop_batch():
    from distgcn_amd.batch import HostBatch
    adjs, wts = _graphs([30, 50, 20], 2)
    adjs[1] = adjs[1].tolil()
    adjs[1][7, 7] = 1
    adjs[1] = adjs[1].tocsr()
    return HostBatch.from_scipy(adjs, wts)


def test_a_faulty_batch_is_reported_by_every_call(engine):
    import torch
    from distgcn_amd import datagen
    from distgcn_amd._lib import DgcnError
    from distgcn_amd.engine import DeviceModel
    hb = _self_loop_batch()
    models = [datagen.random_model(3, 16, seed=s) for s in (1, 2)]
    bank, dm = engine.model_bank(models), DeviceModel(models[0], "cuda:0")
    mog = torch.tensor([0, 1, 1], dtype=torch.int32, device="cuda:0")
    b = engine.upload(hb)
    for _ in range(2):
        with pytest.raises(DgcnError, match="self-loop"):
            engine.forward_bank(b, bank, mog)
    with pytest.raises(DgcnError, match="self-loop"):
        engine.forward(b, dm)
    b = engine.upload(hb)
    for _ in range(2):
        word = torch.zeros(1, dtype=torch.int32, device="cuda:0")
        engine.forward_bank(b, bank, mog, status=word)
        assert int(word) == 1 and int(engine.solve_bank(b, bank, mog)["status"]) == 1 and int(engine.solve(b, dm)["status"]) == 1
    good = engine.upload(_batch_with_columns([30, 50, 20], 2, {})[0])
    for _ in range(2):
        assert int(engine.solve_bank(good, bank, mog)["status"]) == 0 and int(engine.solve(good, dm)["status"]) == 0
        engine.forward_bank(good, bank, mog)


def test_a_captured_pass_reports_its_batch_s_faults(engine):
    import torch
    from distgcn_amd import datagen
    hb = _self_loop_batch()
    bank = engine.model_bank([datagen.random_model(3, 16, seed=s) for s in (1, 2)])
    mog = torch.tensor([0, 1, 1], dtype=torch.int32, device="cuda:0")
    for host, want in ((hb, 1), (_batch_with_columns([30, 50, 20], 2, {})[0], 0)):
        b, word = engine.upload(host), torch.zeros(1, dtype=torch.int32, device="cuda:0")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            engine.forward_bank(b, bank, mog, status=word)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = engine.forward_bank(b, bank, mog, status=word)
        for _ in range(3):
            word.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert int(word) == want
            eager = torch.zeros(1, dtype=torch.int32, device="cuda:0")
            assert torch.equal(out, engine.forward_bank(b, bank, mog, status=eager)) and int(eager) == want
            if not want:
                engine.forward_bank(b, bank, mog)  # (read on the host here: the word the graph reads stays)
