"""GPU: llmhip_kv_plan against the requests served one after the other on the
host. Every value is a whole number and has to be equal."""
import numpy as np
import pytest

import kv_oracle

pytestmark = pytest.mark.gpu


def _run(sampler, page, ring, state, lens, table, T, new=None, release=None, in_place=False, stream=None):
    import torch

    from scriptonait_amd.kv import PagePool

    dev = torch.device("cuda:0")
    i32 = lambda x: torch.tensor(np.asarray(x, dtype=np.int32), device=dev)  # noqa: E731
    R = len(lens)
    pool = PagePool(sampler, len(ring), page, i32(ring), i32(state))
    lens_d, table_d = i32(lens), i32(table)
    out_lens = lens_d if in_place else torch.full_like(lens_d, -9)
    out_state = None if in_place else torch.full((2,), -9, dtype=torch.int32, device=dev)
    granted, start = torch.full((R,), -9, dtype=torch.int32, device=dev), torch.full((R + 1,), -9, dtype=torch.int32, device=dev)
    slots, pos = torch.full((T,), -9, dtype=torch.int64, device=dev), torch.full((T,), -9, dtype=torch.int32, device=dev)
    torch.cuda.synchronize()
    pool.plan(lens_d, table_d, out_lens, granted, start, slots, pos, new_tokens=None if new is None else i32(new),
              release=None if release is None else i32(release), out_free_state=out_state, stream=stream)
    torch.cuda.synchronize()
    if not in_place:
        assert lens_d.tolist() == list(lens) and pool.free_state.tolist() == list(state)
    return dict(lens=out_lens.tolist(), granted=granted.tolist(), start=start.tolist(), slots=slots.tolist(), positions=pos.tolist(),
                table=table_d.tolist(), ring=pool.free_ring.tolist(), state=(pool.free_state if in_place else out_state).tolist())


def _case(seed, R, page, P, mode, tight=False, release=0.1, extra=5):
    rs = np.random.default_rng(seed)
    lens = rs.integers(0, P * page + 1, R)
    gone = (rs.random(R) < release).astype(int)
    new = None
    if mode != "decode":
        new = rs.integers(0, 3 * page + 2, R)
    N = R * P + 7
    order = rs.permutation(N)
    used = -(-lens // page)
    table = np.full((R, P), -12345)  # what is behind a request's pages is nobody's
    at = 0
    for r in range(R):
        table[r, :used[r]] = order[at:at + used[r]]
        at += used[r]
    free = min(N - at, int(R * (0.3 if tight else 3)) + 1)
    head = int(rs.integers(0, N))
    ring = np.full(N, -54321)
    ring[(head + np.arange(free)) % N] = order[at:at + free]
    n = np.where(gone, 0, 1) if new is None else new
    T = int(n.sum()) + extra
    return dict(page=page, ring=ring.tolist(), state=[head, free], lens=lens.tolist(), table=table.tolist(), T=max(T, 0),
                new=None if new is None else new.tolist(), release=gone.tolist())


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("seed,R,page,P,mode,tight,extra", [
    (1, 1, 1, 1, "decode", False, 0), (2, 1, 16, 4, "decode", False, 1), (3, 5, 1, 9, "mixed", False, 3),
    (4, 64, 16, 8, "decode", False, 0), (5, 64, 16, 8, "mixed", True, 0), (6, 63, 24, 5, "mixed", False, -40),
    (7, 1000, 16, 12, "decode", True, 24), (8, 1023, 20, 7, "mixed", False, 100), (9, 1024, 8, 4, "decode", False, 0),
    (10, 1025, 3, 6, "mixed", True, 9), (11, 2500, 16, 3, "mixed", False, 1), (12, 3001, 7, 5, "mixed", True, -500),
    (13, 40, 128, 64, "mixed", False, 10), (14, 7, 256, 300, "mixed", False, 2), (15, 5000, 16, 3, "mixed", False, 77)])
def test_plan_is_the_requests_in_order(sampler, seed, R, page, P, mode, tight, extra, in_place):
    c = _case(seed, R, page, P, mode, tight, extra=extra)
    want = kv_oracle.plan(**c)
    got = _run(sampler, in_place=in_place, **c)
    for name in want:
        assert got[name] == want[name], name
    assert sampler.status().flags == 0


def test_edges(sampler):
    full = dict(page=4, ring=[2, 3, 0, 1], state=[1, 0], lens=[8, 8], table=[[0, 1], [2, 3]], T=2)
    got = _run(sampler, **full)  # no page is free and both tables are full
    assert got["granted"] == [0, 0] and got["slots"] == [-1, -1] and got["start"] == [0, 1, 2] and got["state"] == [1, 0]
    # A request that the pages do not reach for stops later ones, unless they need none.
    c = dict(page=4, ring=[5, 6, 7, 0, 0, 0, 0, 0], state=[0, 3], lens=[4, 4, 1, 4], table=[[0, -1, -1, -1], [1, -1, -1, -1],
             [2, -1, -1, -1], [3, -1, -1, -1]], T=20, new=[5, 8, 2, 1])
    want = kv_oracle.plan(**c)
    assert want["granted"] == [5, 0, 2, 0]
    got = _run(sampler, **c)
    assert all(got[k] == want[k] for k in want)
    # Released and prompted anew in one call: old pages go back, new ones come.
    c = dict(page=2, ring=[9, 8, 7, 0, 0, 0, 0, 0, 0, 0], state=[0, 3], lens=[4, 3], table=[[1, 2, -1], [3, 4, -1]], T=6,
             new=[5, 1], release=[1, 0])
    want = kv_oracle.plan(**c)
    assert want["table"] == [[9, 8, 7], [3, 4, -1]] and want["ring"][3:5] == [1, 2]
    for in_place in (False, True):
        got = _run(sampler, in_place=in_place, **c)
        assert all(got[k] == want[k] for k in want)
    # No request, no token.
    got = _run(sampler, page=4, ring=[0], state=[0, 1], lens=[], table=np.zeros((0, 3)), T=3)
    assert got["start"] == [0] and got["slots"] == [-1] * 3 and got["positions"] == [0] * 3 and got["state"] == [0, 1]
    got = _run(sampler, page=4, ring=[0], state=[0, 1], lens=[0], table=[[-1]], T=0)
    assert got["granted"] == [0] and got["start"] == [0, 1]
    assert sampler.status().flags == 0


@pytest.mark.parametrize("change", [dict(lens=[-1, 2]), dict(lens=[99, 2]), dict(new=[-3, 1]), dict(state=[-1, 3]),
                                    dict(state=[0, 99]), dict(state=[10, 1]), dict(table=[[-7, -7], [1 << 30, -7]], lens=[0, 2]),
                                    dict(ring=[-1, 99, 98, 97])])
def test_bad_values_are_flagged_and_followed_nowhere(sampler, change):
    import torch  # noqa: F401

    from scriptonait_amd.kv import KSTATUS_BAD_INDEX

    c = dict(page=4, ring=[3, 2, 1, 0], state=[0, 2], lens=[0, 2], table=[[-7, -7], [0, -7]], T=4, new=[3, 1])
    c.update(change)
    sampler.status()
    got = _run(sampler, **c)
    assert sampler.status().flags == KSTATUS_BAD_INDEX
    assert all(-1 <= s < 16 for s in got["slots"]) and all(0 <= n <= 8 for n in got["lens"])
    assert 0 <= got["state"][0] < 4 and 0 <= got["state"][1] <= 4


def test_sums_past_31_bits_stop_there(sampler):
    most = 2**31 - 1
    c = dict(page=4, ring=[3, 2, 1, 0], state=[0, 4], lens=[0, 0, 0, 0], table=[[-7, -7]] * 4, T=6, new=[2, most, most, 1])
    got = _run(sampler, **c)
    assert got["start"] == [0, 2, most, most, most] and got["granted"] == [2, 0, 0, 0]
    assert got["slots"] == [12, 13, -1, -1, -1, -1] and got["state"] == [1, 3]
    assert sampler.status().flags == 0


def test_released_pages_outside_the_pool_are_flagged(sampler):
    from scriptonait_amd.kv import KSTATUS_BAD_INDEX

    c = dict(page=4, ring=[3, 2, 1, 0], state=[0, 1], lens=[8, 3], table=[[1, 4], [0, -7]], T=2, release=[1, 0])
    sampler.status()
    got = _run(sampler, **c)
    assert sampler.status().flags == KSTATUS_BAD_INDEX
    assert got["ring"][1:3] == [1, 4] and got["state"] == [0, 3] and got["slots"] == [3, -1]
    c["table"] = [[1, 2], [0, -7]]
    _run(sampler, **c)
    assert sampler.status().flags == 0


def test_outputs_over_inputs_are_refused(sampler):
    import torch

    from scriptonait_amd.kv import PagePool
    from scriptonait_amd.sampler import SamplerError

    x = torch.zeros(64, dtype=torch.int32, device="cuda")
    pool = PagePool(sampler, 8, 16)
    table = torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    slots = torch.zeros(4, dtype=torch.int64, device="cuda")
    args = dict(lens=x[:4], out_lens=x[4:8], granted=x[8:12], start=x[12:17], slots=slots, positions=x[20:24],
                new_tokens=x[24:28], release=x[28:32], table=table)
    for change in [dict(granted=x[24:28]), dict(granted=x[2:6]), dict(start=x[28:33]), dict(start=x[20:25], lens=x[24:28]),
                   dict(out_lens=x[31:35]), dict(out_lens=x[3:7]), dict(out_lens=x[24:28])]:
        with pytest.raises(SamplerError, match="overlap"):
            pool.plan(**{**args, **change})
    pool.plan(**args)
    pool.plan(**{**args, "out_lens": args["lens"]})
    assert sampler.status().flags == 0


def test_other_stream(sampler):
    import torch

    c = _case(21, 300, 16, 9, "mixed")
    got = _run(sampler, stream=torch.cuda.Stream(), **c)
    want = kv_oracle.plan(**c)
    assert all(got[k] == want[k] for k in want)
