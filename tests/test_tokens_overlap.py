"""sort_tokens refuses buffers that overlap: its launches count the slots twice and write
where the counts say.  On the CPU: no call here reaches the device."""
import itertools

import pytest
import torch

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
