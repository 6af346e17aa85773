"""Gradients of the energy in the weights of the last interaction's linears, and the run they are for: gradients, AdamW, the force
field with the new weights."""
import dataclasses
import math

import numpy as np
import pytest
import torch

from oracle import mace_oracle as mo
from oracle import neighbours_oracle as nlo

pytestmark = pytest.mark.gpu


def _case(name):
    from fastmace_b200.model import LARGE, MEDIUM, SMALL, init_weights
    from fastmace_b200.structures import fcc_alloy, nacl
    if name == "large":
        spec = dataclasses.replace(LARGE, avg_num_neighbors=54.0)
        return spec, init_weights(spec, 2), fcc_alloy((2, 2, 2), 0.1, 2)
    spec = SMALL if name == "small" else MEDIUM
    return spec, init_weights(spec, 1), nacl((2, 2, 2) if name != "medium216" else (3, 3, 3), 0.05, 1)


def _energy(spec, weights, s):
    """The oracle's energy in float64, as a function of the weights."""
    snd, rcv, u = nlo.build(s.positions, s.cell, spec.r_cut, 0.0)
    pos, cell = torch.tensor(s.positions, dtype=torch.float64), torch.tensor(s.cell, dtype=torch.float64)
    snd, rcv = torch.as_tensor(snd, dtype=torch.int64), torch.as_tensor(rcv, dtype=torch.int64)
    vectors = pos[rcv] - pos[snd] + torch.as_tensor(u, dtype=torch.float64) @ cell
    species = torch.as_tensor(np.asarray(s.numbers), dtype=torch.int64) - 1
    sh, feats = mo.spherical_harmonics(vectors), mo.bessel_cutoff(torch.linalg.norm(vectors, dim=1), spec)
    h = (weights["emb"][species] / math.sqrt(spec.num_elements))[:, None, :]
    energy = 0.0
    for t in range(spec.num_interactions):
        message, sc = mo.interaction(spec, weights, t, h, species, snd, rcv, sh, feats)
        h = mo.product(spec, weights, t, message, sc, species)
        energy = energy + mo.readout(spec, weights, t, h).sum()
    return spec.scale * energy


@pytest.mark.parametrize("name", ["small", "medium", "medium216", "large"])
def test_gradients_against_the_oracle(name):
    """Elementwise against float64 autograd. The features and gradients that are multiplied come out of fp32 stages that the force
    tests hold to 2e-5 of their largest value; a product of two and its sum over the atoms keeps 1e-4 of the largest gradient."""
    from fastmace_b200.forcefield import B200ForceField
    spec, weights, s = _case(name)
    ff = B200ForceField(spec, weights, s.numbers, s.cell)
    ff.evaluate(s)
    got = ff.weight_gradients()
    names = ["l1.skip.0"] + [f"l1.up.{l}" for l in range(spec.hidden_lmax + 1)]
    assert sorted(got) == sorted(names)
    w64 = {k: v.double().requires_grad_(k in names) for k, v in weights.items()}
    ref = torch.autograd.grad(_energy(spec, w64, s), [w64[k] for k in names])
    present = sorted(set(int(z) - 1 for z in s.numbers))
    for k, r in zip(names, ref):
        g = got[k].double().cpu()
        assert g.shape == r.shape == weights[k].shape
        assert float((g - r).abs().max()) <= 1e-4 * float(r.abs().max()), (k, float((g - r).abs().max() / r.abs().max()))
        if "skip" in k:
            absent = [z for z in range(spec.num_elements) if z not in present]
            assert bool((g[:, absent] == 0).all())


def test_gradients_against_differences():
    """Along random directions of each tensor, central differences of the oracle's float64 energy: the step's third-order error is
    1e-6 of the derivative at most for steps of 1e-4 of weights of order 1, far below the 1e-4 asked above."""
    from fastmace_b200.forcefield import B200ForceField
    spec, weights, s = _case("medium")
    ff = B200ForceField(spec, weights, s.numbers, s.cell)
    ff.evaluate(s)
    g = torch.Generator().manual_seed(1)
    w64 = {k: v.double() for k, v in weights.items()}
    for k, got in ff.weight_gradients().items():
        got = got.double().cpu()
        direction = torch.randn(got.shape, generator=g, dtype=torch.float64)
        step = 1e-4
        e = [float(_energy(spec, {**w64, k: w64[k] + sign * step * direction}, s)) for sign in (1, -1)]
        by_difference = (e[0] - e[1]) / (2 * step)
        # a random direction's derivative is of the order of the gradient's norm
        assert abs(by_difference - float((got * direction).sum())) <= 2e-4 * float(got.norm()), k


@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_step_and_force_field_together(bits):
    """Two steps of an energy fit: gradient, AdamW on a dictionary of weights, a force field with the new ones. The weights follow
    the formula from these gradients, and the others stay."""
    from fastmace_b200.forcefield import B200ForceField
    from fastmace_b200.optimiser import AdamW
    spec, weights, s = _case("medium")
    trained = {k: v.clone().cuda() for k, v in weights.items() if k.startswith("l1.skip") or k.startswith("l1.up")}
    opt = AdamW(trained, lr=1e-3, weight_decay=0.0, state_bits=bits)
    energies = []
    for step in range(2):
        ff = B200ForceField(spec, {**weights, **{k: v.cpu() for k, v in trained.items()}}, s.numbers, s.cell)
        energies.append(ff.evaluate(s)[0])
        grads = ff.weight_gradients()
        old = {k: v.clone() for k, v in trained.items()}
        before = {k: opt.moments(k) for k in trained}
        opt.step(grads)
        for k, g in grads.items():
            m = 0.9 * before[k][0].double() + 0.1 * g.double()
            v = 0.999 * before[k][1].double() + 0.001 * g.double() ** 2
            moved = 1e-3 / (1 - 0.9 ** (step + 1)) * m / (v.sqrt() / math.sqrt(1 - 0.999 ** (step + 1)) + 1e-8)
            tol = 2.0 ** -20 * moved.abs() + 2.0 ** -23 * old[k].double().abs()
            assert bool(((old[k].double() - moved - trained[k].double()).abs() <= tol).all()), k
    assert opt.steps == 2 and all(math.isfinite(e) for e in energies) and energies[0] != energies[1]


def test_refusals():
    from fastmace_b200 import _lib
    from fastmace_b200.forcefield import B200ForceField
    spec, weights, s = _case("small")
    ff = B200ForceField(spec, weights, s.numbers, s.cell)
    with pytest.raises(_lib.Fmb200Error, match="no force call"):
        ff.weight_gradients()
    part = B200ForceField(spec, weights, s.numbers, s.cell, n_owned=10, n_inner=20)
    part.evaluate(s)
    with pytest.raises(_lib.Fmb200Error, match="own all"):
        part.weight_gradients()


@pytest.mark.parametrize("change", ["fewer", "more", "others"])
def test_a_workspace_without_a_call_of_these_atoms_is_refused(change):
    """After ``set_atoms`` (with and without new buffers) the features are those of other atoms, or zeros."""
    from fastmace_b200 import _lib
    from fastmace_b200.forcefield import B200ForceField
    spec, weights, s = _case("small")
    ff = B200ForceField(spec, weights, s.numbers, s.cell)
    ff.evaluate(s)
    before = ff.weight_gradients()
    numbers = {"fewer": s.numbers[:-2], "more": np.concatenate([s.numbers, s.numbers[:2]]), "others": s.numbers[::-1].copy()}[change]
    positions = np.concatenate([s.positions, s.positions[:2] + 1.3])[:len(numbers)]
    ff.set_atoms(numbers)
    with pytest.raises(_lib.Fmb200Error, match="no force call"):
        ff.weight_gradients()
    x = torch.as_tensor(positions, device="cuda")
    ff.rebuild(x)
    ff.compact(x)
    with pytest.raises(_lib.Fmb200Error, match="no force call"):
        ff.weight_gradients()
    ff(x)
    ff.check_status()
    fresh = B200ForceField(spec, weights, numbers, s.cell, positions=x)
    fresh(x)
    for (k, a), b, old in zip(ff.weight_gradients().items(), fresh.weight_gradients().values(), before.values()):
        # the same sums of the same terms, in an order that may follow the buffers' sizes
        assert float((a - b).norm()) <= 1e-5 * float(b.norm()) and not torch.equal(a, old), k


def test_buffers_made_anew_hold_no_call():
    """A list that outgrows its capacity moves every buffer."""
    from fastmace_b200 import _lib
    from fastmace_b200.forcefield import B200ForceField
    spec, weights, s = _case("small")
    at = np.arange(len(s.numbers))
    far = torch.zeros(len(at), 3, dtype=torch.float64, device="cuda")                # pairs far from one another
    far[:, 2] = torch.as_tensor(40.0 * (at // 2) + 2.5 * (at % 2), device="cuda")
    ff = B200ForceField(spec, weights, s.numbers, np.diag([30.0, 30.0, 40.0 * len(s.numbers)]), positions=far)
    ff(far)
    ff.weight_gradients()
    near = torch.as_tensor(s.positions, device="cuda")
    assert ff.rebuild(near)
    with pytest.raises(_lib.Fmb200Error, match="no force call"):
        ff.weight_gradients()


def test_products_that_gave_up_waiting_are_reported():
    """The products' status word as a kernel whose wait has run out leaves it."""
    from fastmace_b200 import _lib, grouped
    from fastmace_b200.forcefield import B200ForceField
    spec, weights, s = _case("small")
    ff = B200ForceField(spec, weights, s.numbers, s.cell)
    ff.evaluate(s)
    good = ff.weight_gradients()
    grouped._status[ff.device.index].fill_(_lib.STATUS_TENSOR_TIMEOUT)
    with pytest.raises(_lib.Fmb200Error, match="gave up waiting"):
        ff.weight_gradients()
    assert all(torch.equal(a, b) for a, b in zip(good.values(), ff.weight_gradients().values()))


def test_captured_with_the_force_call():
    """One graph of force call and gradients, replayed at other positions, gives the bits of the calls one by one."""
    from fastmace_b200 import grouped
    from fastmace_b200.forcefield import B200ForceField
    spec, weights, s = _case("medium")
    ff = B200ForceField(spec, weights, s.numbers, s.cell)
    ff.evaluate(s)
    ff.weight_gradients()
    x = torch.as_tensor(s.positions, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ff(x)
        captured = ff.weight_gradients()
    g = torch.Generator(device="cuda").manual_seed(1)
    for _ in range(2):
        x.add_(0.01 * torch.randn(x.shape, generator=g, device="cuda", dtype=torch.float64))
        ff.compact(x)
        graph.replay()
        torch.cuda.synchronize()
        seen = {k: v.clone() for k, v in captured.items()}
        ff(x)
        for k, v in ff.weight_gradients().items():
            assert torch.equal(seen[k], v), k
    grouped.check_status()
    ff.check_status()


def _close(got, ref):
    """The same fp32 terms from other kernels, summed in another order: 1e-5 of the norm, as for the forces of those paths."""
    assert list(got) == list(ref)
    for k in ref:
        assert float((got[k].double() - ref[k].double()).norm()) <= 1e-5 * float(ref[k].double().norm()), k


@pytest.mark.parametrize("name", ["small", "medium", "large"])
@pytest.mark.parametrize("chunk,edge_adjoint,mirror", [(37, None, True), (1000, None, True), (37, False, True), (1000, False, True),
                                                       (1000, False, False), (None, None, False)])
def test_other_paths_leave_the_same_gradients(name, chunk, edge_adjoint, mirror):
    """Lists in chunks, sender gradients of one chunk at a time, every edge from both ends; atoms without neighbours among them."""
    from fastmace_b200.forcefield import B200ForceField
    from fastmace_b200.model import SPECS, init_weights
    spec = SPECS[name]
    weights = init_weights(spec, 4)
    rng = np.random.default_rng(5)
    edge = (150 * 50.0) ** (1 / 3)
    cell, positions = np.diag([edge, edge, edge + 30.0]), rng.uniform(0, edge, (150, 3))
    positions[[0, 70, 149], :] = [[1, 1, edge + 15.0], [1, 9, edge + 15.0], [9, 1, edge + 15.0]]
    numbers, x = rng.choice([11, 17], 150), torch.tensor(positions, device="cuda")
    whole = B200ForceField(spec, weights, numbers, cell, positions=x)
    whole(x)
    ff = B200ForceField(spec, weights, numbers, cell, positions=x, chunk_edges=chunk, edge_adjoint=edge_adjoint)
    if not mirror:
        ff.work.mirror, ff.work.edge_q, ff.work.edge_dx = None, None, None
    for _ in range(2):
        ff(x)
        ff.check_status()
        _close(ff.weight_gradients(), whole.weight_gradients())


@pytest.mark.parametrize("mode", ["checked", "graph"])
@pytest.mark.parametrize("repeat", [(2, 2, 2), (4, 4, 3)])
def test_gradients_after_the_steps_of_an_engine(mode, repeat):
    """The last force call is that of the last step, captured or not; 384 atoms take the kernels with the radial layer on the SM."""
    from fastmace_b200.engine import B200Engine
    from fastmace_b200.forcefield import B200ForceField
    from fastmace_b200.langevin import IntegratorConfig, Langevin
    from fastmace_b200.model import MEDIUM, init_weights
    from fastmace_b200.state import SimulationState
    from fastmace_b200.structures import nacl
    s = nacl(repeat, 0.05, 1)
    weights = init_weights(MEDIUM, 1)
    ff = B200ForceField(MEDIUM, weights, s.numbers, s.cell)
    state = SimulationState.from_structure(s.with_velocities(300.0, 2), "cuda", seed=3)
    engine = B200Engine(ff, Langevin(state, IntegratorConfig(), temperature_K=300.0), state, mode=mode)
    for steps in (1, 7):
        engine.run(steps)
        fresh = B200ForceField(MEDIUM, weights, s.numbers, s.cell, positions=state.positions)
        fresh(state.positions)
        _close(ff.weight_gradients(), fresh.weight_gradients())
