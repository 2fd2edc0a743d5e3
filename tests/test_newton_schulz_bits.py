"""Which products of a Newton-Schulz iteration take both parts, seen in the workspace: those need 8 bytes a value of X and of A and B, those of the first
parts 6 and 4."""
import ctypes

import pytest

from oztt_amd import device as ozd
from oztt_amd import hip


def asked(desc):
    return hip().oz_orthogonalize_workspace(None, ctypes.byref(desc))


def test_orthogonalize():
    size = 1024, 2048
    one, both = asked(ozd.orthogonalize_desc(*size)), asked(ozd.orthogonalize_desc(*size, exact=True))
    assert one < 8 * 1024 * 2048 + 8 * 1024**2 <= both
    assert both == asked(ozd.orthogonalize_desc(*size, type="f32")) == asked(ozd.orthogonalize_desc(*size, type="f16"))
    small = 512, 2048
    assert asked(ozd.orthogonalize_desc(*small)) == asked(ozd.orthogonalize_desc(*small, exact=True))


@pytest.mark.parametrize("exact", [0, 1, 2, 3])
def test_muon(exact):
    """Each size by its own bit."""
    p = ozd.MuonPlan()
    p.memory, p.count, p.shapes = 256, 3, 2
    p.shape[0], p.shape[1] = ozd.MuonShape(1024, 1024, 1, 0), ozd.MuonShape(2048, 1024, 2, 1)
    p.exact = exact
    want = sum(asked(ozd.orthogonalize_desc(r, c, n, exact=bool(exact >> k & 1))) for k, (r, c, n) in enumerate(((1024, 1024, 1), (2048, 1024, 2))))
    assert hip().oz_muon_workspace(None, ctypes.byref(p)) == want
