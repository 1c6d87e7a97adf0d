"""Work descriptions from what is no GPU tensor: refused with the library's own error."""
import numpy as np
import pytest

import redline_amd as ra


@pytest.mark.parametrize("bad,text", [(None, "must not be None"), ([0, 1], "torch.Tensor"),
                                      (np.zeros(2, np.int32), "torch.Tensor")])
def test_not_a_tensor(bad, text):
    pytest.importorskip("torch")
    from redline_amd import kernels as K
    with pytest.raises(ra.Error, match=text):
        K.decode_work(bad, bad, 2, 1)
    with pytest.raises(ra.Error, match=text):
        K.prefill_work(bad, bad, bad, bad, 2, 1)
