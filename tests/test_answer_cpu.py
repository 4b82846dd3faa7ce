"""What the operators between hidden states and log probabilities refuse without a device."""
import numpy as np
import pytest

from yaxus_b200 import _lib


def test_null_contexts_are_rejected():
    L = _lib.cuda_lib()
    ids = np.zeros(1, np.uint32)
    assert L.yx_matmul_epilogue(None, None, 0, None, None, 0, None, 1, 1, 1, None, 0) == _lib.YX_ERR_INVALID
    assert L.yx_logprob_rows(None, None, 0, 1, 1, 1, ids.ctypes.data, 1, 0, None, None, None, None) == _lib.YX_ERR_INVALID
    assert L.yx_matmul_logprobs(None, None, 0, None, 1, 1, 1, ids.ctypes.data, None, None) == _lib.YX_ERR_INVALID


def test_token_ids_do_not_wrap_around():
    from yaxus_b200.backend import _token_ids
    assert _token_ids([1, 2]).dtype == np.uint32 and _token_ids(np.zeros((0, 3))).shape == (0, 3)
    for wrong in ([-1], np.array([2 ** 32]), [0.5]):
        with pytest.raises(AssertionError):
            _token_ids(wrong)


def test_the_header_s_names_are_the_binding_s():
    import os
    import re
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "yaxus_cuda.h")).read()
    acts = {m.group(1).lower(): int(m.group(2)) for m in re.finditer(r"YX_ACT_(\w+) = (\d+)", text)}
    assert acts == {k: v for k, v in _lib.ACTIVATIONS.items() if k is not None}
    assert int(re.search(r"#define YX_TOP_MAX (\d+)", text).group(1)) == _lib.TOP_MAX
