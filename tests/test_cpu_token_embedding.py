"""What `tv_scaled_embedding_*` refuses on the host, without a GPU."""
import pytest
import torch

from tracevae_amd import hip


def test_refusals_before_any_launch():
    lib = hip.lib()
    one = 1 << 20                       # never dereferenced: validation fails first

    def fwd(rows=4, dim=8, v=10, wt=0, ot=0, w=one, ws=8, ids=one, out=one, os=8):
        return lib.tv_scaled_embedding_fwd(rows, dim, v, wt, ot, w, ws, ids, -1, 1.0, out, os, None)

    for kw in (dict(rows=-1), dict(dim=0), dict(v=0), dict(wt=3), dict(ot=-1), dict(wt=1, ot=0), dict(wt=1, ot=2),
               dict(wt=2, ot=1), dict(ws=7), dict(os=7), dict(w=None), dict(ids=None), dict(out=None),
               dict(w=one + 2), dict(out=one + 1), dict(ids=one + 4), dict(rows=2 ** 31), dict(v=2 ** 31),
               dict(dim=65537, ws=70000, os=70000), dict(v=2 ** 29 + 1), dict(rows=2 ** 29),
               dict(rows=2 ** 25, dim=1025, ws=1025, os=1025), dict(wt=0, ot=1, out=one + 1)):
        assert fwd(**kw) == -1, kw
        assert b'tv_scaled_embedding_fwd' in lib.tv_last_error()
    assert fwd(rows=0, w=None, ids=None, out=None) == 0

    assert lib.tv_scaled_embedding_bwd_workspace_bytes(128, 8, 10) == 0
    need = lib.tv_scaled_embedding_bwd_workspace_bytes(400, 8, 10)
    assert need > 0

    def bwd(rows=400, dim=8, v=10, wt=0, ot=0, ids=one, dout=one, ds=8, dw=one, ws=one, n=need):
        return lib.tv_scaled_embedding_bwd(rows, dim, v, wt, ot, ids, -1, 1.0, dout, ds, dw, ws, n, None)

    for kw, code in ((dict(rows=-1), -1), (dict(dim=0), -1), (dict(v=0), -1), (dict(wt=1, ot=0), -1), (dict(ids=None), -1),
                     (dict(dout=None), -1), (dict(dw=None), -1), (dict(ws=None), -1), (dict(ds=7), -1),
                     (dict(dw=one + 2), -1), (dict(dout=one + 2), -1), (dict(ws=one + 8), -1), (dict(n=need - 1), -3),
                     (dict(rows=2 ** 31), -1)):
        assert bwd(**kw) == code, kw
    for bad in ((-1, 8, 10), (4, 0, 10), (4, 8, 0), (2 ** 31, 8, 10), (4, 65537, 10), (4, 8, 2 ** 31),
                (2 ** 29, 8, 10), (2 ** 25, 1025, 10), (4, 8, 2 ** 29 + 1)):
        assert lib.tv_scaled_embedding_bwd_workspace_bytes(*bad) == -1
    assert lib.tv_scaled_embedding_bwd_workspace_bytes(0, 8, 10) == 0


def test_operator_needs_the_gpu():
    from tracevae_amd import ops
    with pytest.raises(hip.HipLibraryError):
        ops.scaled_embedding(torch.zeros(4, 4), torch.zeros(2, dtype=torch.int64))
