"""hrf_adamw_multi over tensors without a value, on the CPU: what it refuses before anything is launched."""
FAKE = 1 << 20      # an address that is never followed


def _call(lib, **change):
    a = dict(tensors=FAKE, tile_tensor=None, num_tiles=0, count=2, state_bits=8, exp_avg=None, second=None, exp_avg_scale=None,
             second_scale=None, ctl=FAKE, lr=1e-2, lr_dev=None, beta1=0.9, beta2=0.99, eps=1e-15, weight_decay=0.0, grad_scale=1.0,
             max_norm=0.0, norm=None, flags=None, scaler=None, seed=0, zero_grad=0, stream=None)
    a.update(change)
    return lib.hrf_adamw_multi(*a.values())


def test_empty_tensors_need_their_counters():
    from humanrf_amd import _lib
    lib = _lib.lib()
    assert _call(lib, ctl=None) != 0 and b"NULL" in lib.hrf_last_error()
    assert _call(lib, tensors=None, ctl=None) == 0 and _call(lib, count=0) == 0
    for missing in ("tile_tensor", "exp_avg", "second", "ctl"):
        assert _call(lib, **{"num_tiles": 1, "state_bits": 32, "tile_tensor": FAKE, "exp_avg": FAKE, "second": FAKE, missing: None}) != 0
        assert b"NULL" in lib.hrf_last_error()
