"""RMS norm's gradient over the values that it is made from is refused: workgroups that make the
weight's gradient may read them when others have written dx.  CPU only."""
import pytest

from test_bucket_layer_ops import FAKE, refused, rms_back

OTHER = 1 << 20


@pytest.mark.parametrize("place", ["dy", "total"])
def test_dx_over_an_input(place):
    apart = dict(dy=OTHER, total=2 * OTHER, dt=3 * OTHER, dx=4 * OTHER)
    for dw in (FAKE, None):
        refused(rms_back(**{**apart, "dx": apart[place], "dw": dw}), b"dx must not be")
    refused(rms_back(**{**apart, "dx": apart["dt"], "dxs": 17}), b"in place")  # over dtotal it may be
