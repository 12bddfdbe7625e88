"""device.Adapters: arrays that do not belong together are refused in front of the first upload -- no GPU."""
import numpy as np
import pytest

from managedllama2_amd.device import Adapters


@pytest.mark.parametrize("down,up,ranks,scales", [
    ((3, 8, 64), (3, 40, 16), 3, 3), ((3, 8, 64), (2, 40, 8), 3, 3), ((3, 8, 64), (3, 8, 40), 3, 3), ((3, 8, 64), (3, 40, 8), 4, 3),
    ((3, 8, 64), (3, 40, 8), 3, 2), ((3, 512), (3, 40, 8), 3, 3), ((3, 8, 64), (3, 320), 3, 3), ((3, 8, 64), (3, 40, 8), (3, 1), 3)])
def test_arrays_that_do_not_fit_are_refused(down, up, ranks, scales):
    with pytest.raises(ValueError, match="adapters"):
        Adapters.from_host(np.zeros(down), np.zeros(up), np.zeros(ranks), np.zeros(scales))
