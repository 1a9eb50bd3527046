"""Host side of the text encoder's bucket form: its parameters' names and sizes, its refusals (no GPU call)."""
import ctypes

import numpy as np
import pytest

from gradtts_amd import _lib
from gradtts_amd.params import text_encoder_param_shapes
from gradtts_amd.text_encoder import TextEncoder

SIZES = dict(n_vocab=61, n_feats=80, n_channels=160, filter_channels=320, filter_channels_dp=96, n_heads=5, n_layers=2,
             kernel_size=3, n_buckets=16, max_distance=40)


def create(**kw):
    h = ctypes.c_void_p()
    return _lib.lib().gt_text_encoder_create_buckets(*{**SIZES, **kw}.values(), ctypes.byref(h)), h


def test_inventory_matches_params_and_module():
    L = _lib.lib()
    rc, h = create()
    assert rc == 0
    try:
        names = [L.gt_text_encoder_param_name(h, i).decode() for i in range(L.gt_text_encoder_num_params(h))]
        numels = [L.gt_text_encoder_param_numel(h, i) for i in range(L.gt_text_encoder_num_params(h))]
        kw = {k: v for k, v in SIZES.items() if k != "max_distance"}
        shapes = text_encoder_param_shapes(**kw)
        assert names == list(shapes) and numels == [int(np.prod(s)) for s in shapes.values()]
        enc = TextEncoder(61, 80, 160, 320, 96, 5, 2, 3, 0.1, n_buckets=16, max_distance=40)
        assert [(k, tuple(v.shape)) for k, v in enc.state_dict().items()] == list(shapes.items())
        # the training pass keeps nothing of the size of the attention's probabilities
        a, b = (L.gt_text_encoder_train_workspace_bytes(h, 1, t) for t in (2048, 4096))
        assert b < 2.1 * a
    finally:
        L.gt_text_encoder_destroy(h)


@pytest.mark.parametrize("kw", [dict(n_vocab=0), dict(n_channels=512, n_heads=4), dict(n_heads=3), dict(n_heads=0),
                                dict(n_heads=1), dict(kernel_size=2), dict(kernel_size=7), dict(n_layers=0),
                                dict(filter_channels=0), dict(filter_channels_dp=512), dict(n_feats=129),
                                dict(n_buckets=15), dict(n_buckets=2), dict(n_buckets=130), dict(max_distance=4),
                                dict(max_distance=1025)], ids=str)
def test_refusals(kw):
    rc, h = create(**kw)
    assert rc != 0 and not h.value and _lib.lib().gt_last_error()


def test_one_form_of_positions():
    with pytest.raises(ValueError, match="exclude each other"):
        TextEncoder(61, 80, 192, 768, 256, 2, 2, 3, 0.1, 4, n_buckets=32)
    with pytest.raises(ValueError, match="n_buckets"):
        TextEncoder(61, 80, 192, 768, 256, 2, 2, 3, 0.1)
