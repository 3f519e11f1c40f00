"""What `tv_adamw_*` (include/tracevae_hip.h) computes and refuses on the host, without a GPU."""
import ctypes

import pytest
import torch

from tracevae_amd import hip

I64, INT, PTR, DBL = ctypes.c_int64, ctypes.c_int, ctypes.c_void_p, ctypes.c_double


def _plan(sizes, addresses, dtypes=None, decay=None, short=0):
    lib, n = hip.lib(), len(sizes)
    c_sizes = (I64 * n)(*sizes)
    nbytes = lib.tv_adamw_plan_bytes(n, c_sizes)
    image = torch.zeros(max(0, nbytes) // 8 + 8, dtype=torch.int64)
    rc = lib.tv_adamw_plan(n, c_sizes, (INT * n)(*(dtypes or [0] * n)), (PTR * n)(*addresses),
                           (DBL * n)(*(decay or [0.0] * n)), image.data_ptr(), nbytes - short)
    return rc, image


def test_state_and_plan_sizes():
    lib = hip.lib()
    sizes = (I64 * 5)(1, 256, 257, 0, 4097)
    assert lib.tv_adamw_state_elements(5, sizes) == 256 + 256 + 512 + 0 + 4352
    # one entry per started 4096 elements, and one per tensor
    grow = [lib.tv_adamw_plan_bytes(1, (I64 * 1)(n)) for n in (0, 1, 4096, 4097, 8193)]
    assert grow[1] == grow[2] and grow[1] - grow[0] == grow[3] - grow[2] == grow[4] - grow[3] > 0
    assert lib.tv_adamw_state_elements(1, (I64 * 1)(-1)) == -1
    assert lib.tv_adamw_state_elements(2, (I64 * 2)(2 ** 60, 2 ** 60)) == -1
    assert lib.tv_adamw_plan_bytes(1, (I64 * 1)(-1)) == -1
    assert lib.tv_adamw_state_elements(0, None) == -1


def test_plan_refuses():
    lib = hip.lib()
    assert _plan([100, 50], [4096, 8192])[0] == 0
    assert _plan([100, 50], [4096, 4096 + 400])[0] == 0            # side by side
    for args, text in ((([100, 50], [4096, 4096 + 396]), b'overlap'),
                       (([100, 100], [4096, 4096]), b'overlap'),
                       (([50, 100], [4096 + 396, 4096]), b'overlap'),
                       (([100, 50], [4096, 4098]), b'misaligned'),
                       (([100, 50], [4096, None]), b'null'),
                       (([100], [4096], [3]), b'dtype'),
                       (([100], [4096], [0], [-0.5]), b'decay'),
                       (([100], [4096], [0], [float('nan')]), b'decay'),
                       (([100], [4096], [0], [float('inf')]), b'decay')):
        assert _plan(*args)[0] == -1
        assert text in lib.tv_last_error(), text
    assert _plan([100, 0], [4096, None])[0] == 0                   # an empty tensor has no address
    assert _plan([100, 200], [4096, 4296], [1, 2])[0] == 0         # 100 bf16 take 200 bytes
    assert _plan([100], [4096], short=8)[0] == -3                  # plan buffer too small


def test_control_refuses():
    lib = hip.lib()
    image = torch.zeros(lib.tv_adamw_control_bytes() // 8, dtype=torch.int64)
    assert lib.tv_adamw_control(3, 1e-3, 0.5, 0.25, 1e-8, image.data_ptr()) == 0
    f = image.view(torch.float64)
    assert int(image[0]) == 3 and f[1:7].tolist() == [1e-3, 0.5, 0.25, 1e-8, 0.125, 0.015625]
    for bad in ((-1, 1e-3, 0.9, 0.99, 1e-8), (0, -1e-3, 0.9, 0.99, 1e-8), (0, 1e-3, 1.0, 0.99, 1e-8),
                (0, 1e-3, 0.9, 1.0, 1e-8), (0, 1e-3, -0.1, 0.9, 1e-8), (0, 1e-3, 0.9, 0.99, -1.0),
                (0, float('nan'), 0.9, 0.99, 1e-8), (0, float('inf'), 0.9, 0.99, 1e-8),
                (0, 1e-3, 0.9, 0.99, float('inf')), (0, 1e-3, float('nan'), 0.99, 1e-8)):
        assert lib.tv_adamw_control(*bad, image.data_ptr()) == -1, bad
    assert lib.tv_adamw_control(0, 1e-3, 0.9, 0.99, 1e-8, None) == -1


def test_control_has_the_products_that_the_steps_form():
    """beta^step as a product of `step` factors, bit for bit, while 1 - beta^step shows it."""
    for step in (0, 1, 2, 37, 5000, 100000, 10 ** 12):
        image = torch.zeros(hip.lib().tv_adamw_control_bytes() // 8, dtype=torch.int64)
        assert hip.lib().tv_adamw_control(step, 1e-3, 0.9, 0.999, 1e-8, image.data_ptr()) == 0
        got = image.view(torch.float64)[5:7].tolist()
        want = [1.0, 1.0]
        for _ in range(min(step, 100000)):
            want = [want[0] * 0.9, want[1] * 0.999]
        for x, y in zip(got, want):
            assert x == y or (x <= 1e-30 and y <= 1e-30)
        assert int(image[0]) == step


def test_step_refuses_before_any_launch():
    lib = hip.lib()
    one = 1 << 20                       # never dereferenced: validation fails first
    _, plan = _plan([100, 50], [4096, 8192], [0, 1])
    grads = (PTR * 2)(4096, 8192)
    wsb = lib.tv_adamw_workspace_bytes(2)

    def call(plan=plan.data_ptr(), dev=one, g=grads, bits=32, m=one, v=one, s1=None, s2=None, master=one,
             control=one, clip=1.0, norm=None, guard=None, kind=0, host=None, ws=one, n=wsb):
        return lib.tv_adamw_step(plan, dev, g, bits, m, v, s1, s2, master, control, clip, norm, 0, guard,
                                 kind, host, ws, n, None)

    empty = torch.zeros(64, dtype=torch.int64)
    for kw, code in ((dict(plan=None), -1), (dict(dev=None), -1), (dict(g=None), -1), (dict(control=None), -1),
                     (dict(plan=empty.data_ptr()), -1), (dict(bits=16), -1), (dict(m=None), -1),
                     (dict(v=None), -1), (dict(bits=8), -1), (dict(m=one + 4), -1), (dict(master=None), -1),
                     (dict(master=one + 8), -1), (dict(clip=-1.0), -1), (dict(clip=float('nan')), -1),
                     (dict(clip=0.0, norm=one), -1), (dict(guard=one), -1), (dict(kind=1), -1),
                     (dict(kind=3, guard=one), -1), (dict(host=one), -1), (dict(ws=None), -1),
                     (dict(n=wsb - 8), -3), (dict(g=(PTR * 2)(4097, 8192)), -1),
                     (dict(g=(PTR * 2)(4096, 8193)), -1)):
        assert call(**kw) == code, kw


def test_optimizer_needs_the_gpu():
    from tracevae_amd import AdamW
    with pytest.raises(hip.HipLibraryError):
        AdamW([torch.zeros(4)])


def test_weight_decay_is_a_field_of_the_configuration():
    from tracevae_amd.config import ExpConfig, config_from_dict, config_to_dict, parse_flags
    c = ExpConfig()
    assert c.train.optimizer == 'rmsprop' and c.train.weight_decay == 0.01
    parse_flags(c, ['--train.optimizer=adamw8', '--train.weight_decay=0.1'])
    d = config_to_dict(c)
    assert d['train']['weight_decay'] == 0.1
    del d['train']['weight_decay']                       # a configuration saved before it existed
    assert config_from_dict(ExpConfig(), d).train.weight_decay == 0.01
