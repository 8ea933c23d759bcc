"""sort_tokens refuses buffers that overlap (on the CPU: no call that is refused reaches the
device), except rows in place of ids."""
import itertools

import pytest
import torch

import tokens_ref as ref

P = 1 << 24  # addresses that no call may read
NAMES = ("ids", "w", "off", "slots", "rows", "ws")


@pytest.fixture(scope="module")
def cl():
    import cascadia_amd

    return cascadia_amd


@pytest.mark.parametrize("T,k,E", [(4, 2, 8), (9000, 8, 384), (1 << 20, 16, 1024)])
def test_overlapping_buffers_are_refused(cl, T, k, E):
    L, arg = cl.lib(), cl._lib.ERR_ARG
    need = L.cascadia_int4_sort_tokens_workspace_bytes(T, k, E)
    size = dict(ids=4 * T * k, w=4 * T * k, off=4 * (E + 1), slots=4 * T * k, rows=4 * T * k, ws=need)
    far = {n: (i + 1) * 16 * P for i, n in enumerate(NAMES)}

    def call(**kw):
        a = dict(far, **kw)
        return L.cascadia_int4_sort_tokens(a["ids"], a["w"], 0.0, T, k, E, a["off"], a["slots"],
                                           a["rows"], a["ws"], None)

    for x, y in itertools.combinations(NAMES, 2):
        if {x, y} == {"ids", "w"} or not (size[x] and size[y]):
            continue  # (both only read)
        at = far[x]
        last = at + (size[x] - 4) // 16 * 16  # (workspaces lie on 16 bytes)
        for where in (at, last, at - (size[y] - 4) // 16 * 16):
            if {x, y} == {"ids", "rows"} and where == at:
                continue  # (rows may be ids)
            assert call(**{y: where}) == arg, (x, y, where - at)


@pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are none of the device's")
def test_neighbours_are_not_refused(cl):
    """Parts of one buffer, one behind the other, and an id buffer that is the weights'."""
    L, arg = cl.lib(), cl._lib.ERR_ARG
    for T, k, E in ((4, 2, 8), (9000, 8, 384)):
        n, off = 4 * T * k, 4 * (E + 1)
        at = [P, P + n, P + n + off, P + 2 * n + off, P + 3 * n + off]
        ids, o, slots, rows, w = at
        assert L.cascadia_int4_sort_tokens(ids, w, 0.0, T, k, E, o, slots, rows, None, None) != arg
        assert L.cascadia_int4_sort_tokens(ids, ids, 0.0, T, k, E, o, slots, rows, None, None) != arg


@pytest.mark.gpu
@pytest.mark.parametrize("T,k,E", [(1, 1, 1), (100, 8, 60), (3000, 2, 5), (9000, 8, 384),
                                   (70001, 8, 1024), (200000, 3, 17)])
def test_rows_in_place_of_ids(cl, T, k, E):
    g = torch.Generator()
    g.manual_seed(T)
    ids = torch.randint(-1, E + 1, (T, k), generator=g, dtype=torch.int32)
    want = ref.sort(ids.numpy(), E)
    rows = ids.cuda()
    off, slots = (torch.empty(n, dtype=torch.int32, device="cuda") for n in (E + 1, T * k))
    cl.sort_tokens(rows, k, E, off, slots, rows)
    for a, b in zip((off, slots, rows), want):
        assert torch.equal(a.cpu(), torch.from_numpy(b))
