"""What the paged cache and the int8-activation entries refuse on the host: calls that would reach past their buffers or whose
sizes pass what the kernels count in."""
import pytest

I, N = -22, -95


def _attn(L, nitems, nown, parts, ws):
    return L.ecd_paged_attn(16, 512, 16, 16, 8, 4, 8, 8, ws, 16, 8, nitems, nown, parts, 1, 4, 2, 1, 4, 9, 4, 2, 16, 128, 0.1, None)


@pytest.mark.parametrize("nitems,nown,parts,ws", [(1, 1, 1, None), (1, 1, 1, 16), (3, 4, 4, 16), (1, 2, 2, 16)])
def test_shared_parts_need_places_of_their_own(nitems, nown, parts, ws):
    """Shared parts with as many parts as a row's own slots have: they would be written to the own parts' places, or to a
    workspace that is not there."""
    from estudiocanciones_amd import _ffi
    assert _attn(_ffi.lib(), nitems, nown, parts, ws) == I
