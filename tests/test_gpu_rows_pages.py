"""The row operators, the page pool and the table in one program: a decode step
with branches. Keys of each new token are looked up, their rows summed with
weights to the token's row, the rows written to the tokens' pages, the pages
shared by branches, moved and let go. Everything a sequence holds is compared
with what was written for it, kept on the host in 64 bits."""
import numpy as np
import pytest
import torch

import hkv_b200 as H

pytestmark = pytest.mark.gpu

DIM, SIZE, PAGES, ROWS, WIDTH, SLOTS = 24, 4, 96, 12, 10, 3
U = 2.0 ** -24


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def test_decode_steps_with_branches():
    rng = np.random.default_rng(5)
    table = H.HashTable(H.EvictStrategy.kLru)
    table.init(H.HashTableOptions(init_capacity=4096, max_capacity=4096,
                                  max_hbm_for_vectors=1 << 30, dim=DIM))
    values = torch.from_numpy(rng.standard_normal((3001, DIM)).astype(np.float32)).cuda()
    keys = torch.arange(1, 3001, device="cuda")
    table.insert_or_assign(3000, keys, values[1:].contiguous())
    plane = torch.zeros((PAGES, SIZE, DIM), device="cuda")
    pool = H.PagePool([plane], SIZE, ROWS, WIDTH)
    cache = plane.view(PAGES * SIZE, DIM)
    held = {r: [] for r in range(ROWS)}  # row -> (sum, sum of magnitudes) of each token

    def write(rows):
        """One new token for each of the rows, as a decode step takes it."""
        n = len(rows)
        picked = rng.integers(1, 3001, (n, SLOTS))
        weights = rng.standard_normal((n, SLOTS)).astype(np.float32)
        picked[0, 1] = 5000  # a key that the table lacks
        asked = torch.from_numpy(picked).cuda()
        found = torch.zeros(n * SLOTS, dtype=torch.bool, device="cuda")
        looked_up = torch.full((n * SLOTS, DIM), float("nan"), device="cuda")
        table.find(n * SLOTS, asked, looked_up, found)
        places = torch.arange(n * SLOTS, device="cuda", dtype=torch.int32)
        places = torch.where(found, places, -1).view(n, SLOTS)
        tokens = torch.zeros((n, DIM), device="cuda")
        H.combine_rows(n, looked_up, places, torch.from_numpy(weights).cuda(), tokens)
        who, status = i32(rows), torch.zeros(n, dtype=torch.bool, device="cuda")
        at = pool.lengths[who.long()].long()
        pool.resize(n, who, (at + 1).to(torch.int32), status)
        assert status.all()
        page = pool.table[who.long(), at // SIZE].long()
        positions = (page * SIZE + at % SIZE).to(torch.int32).view(n, 1)
        H.dispatch_rows(n, tokens, positions, cache)
        known = np.where(picked < 3001, picked, 0)
        terms = weights[..., None].astype(np.float64) * values.double().cpu().numpy()[known]
        terms[picked >= 3001] = 0
        for k, r in enumerate(rows):
            held[r].append((terms[k].sum(0), np.abs(terms[k]).sum(0)))

    def check():
        torch.cuda.synchronize()
        lengths, entries, got = pool.lengths.tolist(), pool.table.cpu().numpy(), plane.cpu().numpy()
        counts = np.zeros(PAGES, int)
        for r in range(ROWS):
            assert lengths[r] == len(held[r])
            pages = entries[r, :-(-lengths[r] // SIZE)]
            np.add.at(counts, pages, 1)
            for k, (want, mass) in enumerate(held[r]):
                # slots fused multiply-adds in float32
                assert (np.abs(got[pages[k // SIZE], k % SIZE] - want) <= SLOTS * U * mass).all()
        assert (pool.refs.cpu().numpy() == counts).all()

    for step in range(40):
        live = [r for r in range(ROWS) if held[r]] or [0]
        if not held[0]:
            write([0])
            continue
        growing = [r for r in live if len(held[r]) < SIZE * WIDTH - 1][:6]
        if growing:
            write(growing)
        if step % 3 == 0:  # two branches take the place of other rows
            src = rng.choice(live, 2).tolist()
            dst = rng.choice([r for r in range(ROWS) if r not in src], 2, replace=False).tolist()
            pool.fork(2, i32(src), i32(dst))
            for s, d in zip(src, dst):
                held[d] = list(held[s])
        if step % 5 == 4:  # tokens taken back, a row given up
            r = int(rng.choice(live))
            keep = int(rng.integers(0, len(held[r]) + 1))
            pool.resize(1, i32([r]), i32([keep]))
            del held[r][keep:]
            gone = int(rng.integers(1, ROWS))
            pool.free(1, i32([gone]))
            held[gone] = []
        if step % 7 == 6:
            pool.compact()
        check()
    table.close()
