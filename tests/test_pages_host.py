"""Refusals of the calls that deal and return pages, on any machine."""
import os

import pytest

from omegalax_amd import _lib
from test_attn_host import BIG, _run

pytestmark = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH),
                                reason="libomx_gdn.so not built (python -m omegalax_amd.build)")

ASSIGN = dict(table=16, N=4, width=10, lengths=16, new=16, free=16, count=16, n_pages=40, page=16, T=30, cu=16, positions=16,
              slots=16, missing=16, ws=None, ws_bytes=0, stream=None)
RELEASE = dict(table=16, N=4, width=10, lengths=16, free=16, count=16, n_pages=40, page=16, window=0, sinks=0, ws=None,
               ws_bytes=0, stream=None)
BAD = [(dict(N=-1), "sequence count"), (dict(N=(1 << 20) + 1), "sequence count"), (dict(page=8), "page size"), (dict(page=24), "page size"),
       (dict(page=1 << 17), "page size"), (dict(n_pages=-1), "page count"), (dict(n_pages=1 << 31), "page count"),
       (dict(width=-1), "block table"), (dict(width=1 << 30), "block table"), (dict(table=None), "NULL"), (dict(lengths=None), "NULL"),
       (dict(free=None), "NULL"), (dict(count=None), "NULL")]


@pytest.mark.parametrize("over,msg", BAD + [
    (dict(T=-1), "too many tokens"), (dict(T=1 << 31), "too many tokens"), (dict(new=None), "NULL"), (dict(cu=None), "NULL"),
    (dict(positions=None), "NULL"), (dict(slots=None), "NULL"), (dict(missing=None), "NULL"), (dict(N=5000), "workspace"),
    (dict(N=5000, ws=8, ws_bytes=1 << 20), "aligned")])
def test_assign_refuses(over, msg):
    rc, err = _run("omx_gdn_pages_assign", ASSIGN, over)
    assert rc == _lib.EINVAL and msg in err


@pytest.mark.parametrize("over,msg", BAD + [
    (dict(window=-1), "window"), (dict(window=5, sinks=-1), "sinks"), (dict(sinks=1), "sinks"), (dict(width=10000), "workspace"),
    (dict(width=10000, ws=8, ws_bytes=1 << 20), "aligned"), (dict(N=1 << 20, width=1 << 17), "grid too large")])
def test_release_refuses(over, msg):
    rc, err = _run("omx_gdn_pages_release", RELEASE, over)
    assert rc == _lib.EINVAL and msg in err


def test_workspaces():
    L = _lib.lib()
    assert L.omx_gdn_pages_assign_workspace_size(4096) == 0 and L.omx_gdn_pages_assign_workspace_size(4097) > 0
    assert L.omx_gdn_pages_release_workspace_size(64, 512) == 0 and L.omx_gdn_pages_release_workspace_size(64, 513) > 0
    for x in BIG[2:]:
        assert L.omx_gdn_pages_assign_workspace_size(x) == 0
        assert L.omx_gdn_pages_release_workspace_size(x, 10) == 0 and L.omx_gdn_pages_release_workspace_size(10, x) == 0


def test_workspace_of_many_rows():
    """One workgroup returns up to 8,192 rows, whatever their width: more take counts of 4,096 entries each."""
    size = _lib.lib().omx_gdn_pages_release_workspace_size
    for width in (0, 1, 2, 3, 4):
        assert size(8191, width) == size(8192, width) == 0
        entries = 8193 * width
        assert size(8193, width) >= 4 * ((entries + 4095) // 4096 + 1)


def test_an_empty_return_is_no_op():
    assert _run("omx_gdn_pages_release", RELEASE, dict(N=0, table=None, lengths=None))[0] == _lib.OK
    assert _run("omx_gdn_pages_release", RELEASE, dict(width=0, table=None))[0] == _lib.OK


def test_python_checks_before_the_library():
    torch = pytest.importorskip("torch")
    import omegalax_amd as om
    t, l, c = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        om.kv_pages_assign(t, l, l, l, c, page_size=16, tokens=3)
    with pytest.raises(ValueError, match="GPU"):
        om.kv_pages_release(t, l, l, c, page_size=16)


def test_the_reference_by_hand():
    from pages_reference import assign, release
    table, free = [[3, -1, -1], [-1, -1, -1], [5, -1, -1]], [0, 1, 2, 4, 9, 9]
    cu, pos, slots, missing, count = assign(table, [10, 0, -1], [8, 17, 4], free, 4, 16, 30)
    assert table == [[3, 4, -1], [2, 1, -1], [5, -1, -1]] and count == 1 and missing == 0
    assert cu == [0, 8, 25, 25] and pos == [*range(10, 18), *range(17), -1, -1, -1, -1, -1]
    assert slots == [*range(58, 64), 64, 65, *range(32, 48), 16, -1, -1, -1, -1, -1]
    assert release(table, [10, 0, -1], free, count, 16) == 4 and free == [0, 1, 2, 4, 9, 9]
    assert table == [[3, -1, -1], [-1, -1, -1], [5, -1, -1]]
