"""The measured cases of perf/operators.py at small sizes: the plain forms (CPU) and
the framework's calls (GPU) against the cases' own definition in 64 bits. Whole
numbers are equal. Floating results may be off by the rounding to their type plus
2^-12 of the largest value: 4096 roundings of a float32 sum of that size, the
longest sum here. That tells a wrong result from a right one; bounds element by
element are in test_gpu_rows.py."""
import importlib.util
import os
import random

import pytest
import torch

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "perf",
                    "operators.py")
spec = importlib.util.spec_from_file_location("operator_cases", PATH)
cases = importlib.util.module_from_spec(spec)
spec.loader.exec_module(cases)


def small(seed):
    rng = random.Random(seed)
    while True:
        case = cases.draw(rng)
        if cases.work(case)["bytes"] < 3e6:
            return case


def compare(case, seed):
    state = cases.prepare(case, seed)
    first = {k: torch.as_tensor(v).clone() for k, v in cases.run(state).items()}
    again = cases.run(state)
    exact = cases.exact(case, seed)
    assert set(first) == set(exact)
    for name, got in first.items():
        assert torch.equal(got, torch.as_tensor(again[name])), (case, name)
        want = torch.as_tensor(exact[name]).to(got.device)
        assert got.shape == want.shape, (case, name)
        if not got.is_floating_point():
            assert torch.equal(got.long(), want.long()), (case, name)
            continue
        slack = (torch.finfo(got.dtype).eps / 2 + 2.0 ** -12) * want.double().abs().max() \
            if want.numel() else 0.0
        assert ((got.double() - want.double()).abs() <= slack).all(), (case, name)


def test_listed_cases():
    listed = cases.listed()
    assert 4 <= len(listed) <= 12 and len({c["name"] for c in listed}) == len(listed)
    assert {c["op"] for c in listed} == {"dispatch", "combine", "copy", "branch", "compact"}
    sizes = [cases.work(c)["bytes"] for c in listed]
    assert max(sizes) >= 16 * min(sizes) > 0


@pytest.mark.skipif(torch.cuda.is_available(), reason="the GPU form of this test runs instead")
@pytest.mark.parametrize("seed", range(12))
def test_plain_forms(seed):
    compare(small(seed), seed)


@pytest.mark.gpu
@pytest.mark.parametrize("own", [False, True])
@pytest.mark.parametrize("seed", range(30))
def test_cases_on_the_gpu(seed, own, monkeypatch):
    monkeypatch.setattr(cases, "own", own)
    compare(small(seed), seed)


def held(state, table):
    """The entries of a page table that mean something."""
    size = state["case"]["page_tokens"]
    pages = (state["lengths"] + size - 1) // size
    return torch.arange(table.shape[1], device=table.device) < pages[:, None]


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["dispatch", "combine", "compact"])
def test_every_pass_writes_its_outputs(op, monkeypatch):
    """A second pass into outputs that were overwritten in between; rows that no place
    has and entries behind a row's pages are left as they then are."""
    monkeypatch.setattr(cases, "own", True)
    seeds = [seed for seed in range(200) if small(seed)["op"] == op][:6]
    assert len(seeds) == 6
    for seed in seeds:
        state = cases.prepare(small(seed), seed)
        out = cases.run(state)
        first = {k: v.clone() for k, v in out.items()}
        for name, t in out.items():
            if name != "planes":
                t.fill_(77)
        again = cases.run(state)
        for name, want in first.items():
            want, got = want, again[name]
            written = torch.ones_like(want, dtype=torch.bool)
            if op == "compact" and name == "table":
                written = held(state, want)
            if name in ("rows", "grad_rows"):
                rows = state["positions"].reshape(-1).long()
                written[:] = False
                written[rows[rows >= 0]] = True
            assert torch.equal(got[written], want[written]), (seed, name)
            assert (got[~written] == 77).all(), (seed, name)
