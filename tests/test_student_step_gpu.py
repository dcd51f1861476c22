"""GPU test of the operators around a network's output as they are used together: a student's training step in float16 -- layer norm, an affine layer with ReLU and its bypass, layer norm, the
output layer, distillation from a teacher's top logits beside the log-probability of a given label with the entropy as a bonus, and the backward pass of all of it -- against the same
network in float64.

Bound.  Every stage rounds to float16 once, moving what it hands on by at most half a step (2^-11) of its size; between the input and a derivative lie at most 12 such stages, and none
of them (rows of unit size after a layer norm, weights of norm below 2, softmax) enlarges a relative difference by more than 4: 12 x 4 x 2^-11 = 2.4 % in the 2-norm."""
import threading
import pytest, torch
from tests.rowop_cases import generator
pytestmark = pytest.mark.gpu
ROWS, DIM, PDFS, TOP, T, EPS = 150, 96, 601, 7, 2.0, 1e-5

def data(seed, dtype=torch.float16):
    g = generator(seed); r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    d = dict(x=r(ROWS, DIM).to(dtype), g1=1 + 0.2 * r(DIM), o1=0.1 * r(DIM), w1=(r(DIM, DIM) * DIM ** -0.5).to(dtype), b1=0.1 * r(DIM), g2=1 + 0.2 * r(DIM), o2=0.1 * r(DIM),
             w2=(r(PDFS, DIM) * 2 * DIM ** -0.5).to(dtype), b2=0.1 * r(PDFS), values=(2 * r(ROWS, TOP)).to(dtype), weights=torch.rand(ROWS, generator=g, device="cuda"))
    d["indexes"] = torch.randint(-1, PDFS, (ROWS, TOP), generator=g, device="cuda").to(torch.int32); d["labels"] = torch.randint(-1, PDFS, (ROWS,), generator=g, device="cuda").to(torch.int32)
    d["advantage"], d["bonus"] = 0.3 * r(ROWS), torch.full((ROWS,), 0.01, device="cuda")
    return d

def step(d):
    """forward and backward; every operator through its public entry point"""
    from kaldi_amd import cumatrix as cm, objective as ob
    h = lambda: torch.empty_like(d["x"]); v = lambda n=ROWS: torch.empty(n, device="cuda")  # noqa: E731
    n1, m1, s1 = h(), v(), v(); cm.LayerNormPerRow(d["x"], d["g1"], d["o1"], EPS, n1, m1, s1)
    a, pre = h(), h(); cm.AffinePerRow(n1, d["w1"], d["b1"], "relu", d["x"], a, pre)
    n2, m2, s2 = h(), v(), v(); cm.LayerNormPerRow(a, d["g2"], d["o2"], EPS, n2, m2, s2)
    z = torch.empty(ROWS, PDFS, dtype=d["x"].dtype, device="cuda"); cm.AffinePerRow(n2, d["w2"], d["b2"], "none", None, z)
    objf, dz = v(), torch.empty_like(z); ob.ComputeDistillObjfAndDeriv(ob.DistillationOptions(T), z, d["values"], d["indexes"], d["weights"], objf, dz)
    lp, ent, stats, alt = v(), v(), torch.empty(ROWS, 2, device="cuda"), torch.empty(ROWS, 3, dtype=torch.int32, device="cuda"); ob.LabelLogProbs(z, d["labels"], lp, ent, stats, None, alt)
    dl = torch.empty_like(z); ob.DiffLabelLogProbs(z, d["labels"], stats, ent, d["advantage"], d["bonus"], dl); dz += dl
    dn2, dw2, db2 = h(), torch.empty_like(d["w2"]), v(PDFS); cm.DiffAffinePerRow(n2, d["w2"], None, "none", dz, dn2, dw2, db2)
    da, dg2, do2 = h(), v(DIM), v(DIM); cm.DiffLayerNormPerRow(a, dn2, d["g2"], m2, s2, da, dg2, do2)
    dn1, dw1, db1 = h(), torch.empty_like(d["w1"]), v(DIM); cm.DiffAffinePerRow(n1, d["w1"], pre, "relu", da, dn1, dw1, db1)
    dx, dg1, do1 = h(), v(DIM), v(DIM); cm.DiffLayerNormPerRow(d["x"], dn1, d["g1"], m1, s1, dx, dg1, do1); dx += da      # the bypass
    return dict(z=z, objf=objf, lp=lp, ent=ent, alt=alt, x=dx, g1=dg1, o1=do1, w1=dw1, b1=db1, g2=dg2, o2=do2, w2=dw2, b2=db2)

def reference(d):
    p = {k: d[k].double().cpu().requires_grad_(True) for k in ("x", "g1", "o1", "w1", "b1", "g2", "o2", "w2", "b2")}
    ln = lambda x, g, o: torch.nn.functional.layer_norm(x, (DIM,), g, o, EPS)  # noqa: E731
    a = torch.relu(ln(p["x"], p["g1"], p["o1"]) @ p["w1"].t() + p["b1"]) + p["x"]; z = ln(a, p["g2"], p["o2"]) @ p["w2"].t() + p["b2"]
    idx = d["indexes"].long().cpu(); used = idx >= 0; t = torch.where(used, d["values"].double().cpu() / T, -1e300); logp = torch.log_softmax(t, 1); pt = logp.exp() * used
    lq = torch.log_softmax(z / T, 1).gather(1, idx.clamp(min=0)); objf = d["weights"].double().cpu() * T * T * (pt * torch.where(used, lq - logp, torch.zeros_like(lq))).sum(1)
    lq1 = torch.log_softmax(z, 1); y = d["labels"].long().cpu(); lp = torch.where(y >= 0, lq1.gather(1, y.clamp(min=0)[:, None])[:, 0], torch.zeros(ROWS, dtype=torch.float64)); ent = -(lq1.exp() * lq1).sum(1)
    (objf.sum() + (d["advantage"].double().cpu() * lp).sum() + (d["bonus"].double().cpu() * ent).sum()).backward()
    return dict(z=z.detach(), objf=objf.detach(), lp=lp.detach(), ent=ent.detach(), **{k: v.grad for k, v in p.items()})

def test_a_students_step_matches_the_network_in_float64():
    d = data(1); got, want = step(d), reference(d)
    for k, w in want.items():
        off = (got[k].double().cpu() - w).norm() / w.norm(); assert off <= 0.024, (k, off.item())
    assert torch.equal(got["alt"][:, 0].long().cpu(), got["z"].float().cpu().argmax(1))

def test_the_step_in_a_graph_and_on_two_threads():
    a, b = data(2), data(3); want = step(a), step(b); torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph): out = step(a)
    first = {k: v.clone() for k, v in a.items()}
    for i in range(3):      # the graph's inputs changed in place between replays, and other eager work beside it
        for k in a: a[k].copy_((b if i % 2 else first)[k])
        torch.cuda.synchronize(); graph.replay(); step(b); torch.cuda.synchronize()
        assert all(torch.equal(out[k], want[i % 2][k]) for k in out), i
    for k in a: a[k].copy_(first[k])
    torch.cuda.synchronize(); got = [None, None]
    def run(i, d):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5): got[i] = step(d)
            torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=run, args=(i, d)) for i, d in enumerate((a, b))]
    for t in threads: t.start()
    for t in threads: t.join()
    assert all(torch.equal(got[i][k], want[i][k]) for i in (0, 1) for k in want[i])
