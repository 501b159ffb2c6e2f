"""The routed products' host side: argument checks before any launch, sizes the
C ABI refuses, and the polynomial check.  No GPU."""

import ctypes

import pytest
import torch

import gmmxx_b200 as gm
from gmmxx_b200 import _native as nat
from gmmxx_b200 import experts


@pytest.fixture
def host_checks(monkeypatch):
    """Let CPU tensors pass the device check: every refusal below comes before a launch."""
    def check(t, name, dtype=None):
        return t.contiguous()

    monkeypatch.setattr(experts, "_check_input", check)


def _groups(n=4, k=3, top=1):
    shape = (n,) if top == 1 else (n, top)
    s = n * top
    return experts.RowGroups(torch.zeros(s, dtype=torch.int32), torch.zeros(k + 1, dtype=torch.int32),
                             torch.zeros(nat.group_tiles_len(s, k), dtype=torch.int32), n, top, k, shape)


def test_public_names():
    for name in ("RowGroups", "group_rows", "grouped_matmul", "grouped_matmul_backward", "orthogonalize"):
        assert name in gm.__all__ and hasattr(gm, name)


def test_host_tensors_are_refused():
    with pytest.raises(ValueError, match="labels: must be on a CUDA device"):
        gm.group_rows(torch.zeros(4, dtype=torch.int64), 3)
    with pytest.raises(ValueError, match="must be on a CUDA device"):
        gm.grouped_matmul(torch.zeros(4, 2), torch.zeros(3, 2, 2), _groups())
    with pytest.raises(ValueError, match="must be on a CUDA device"):
        gm.grouped_matmul_backward(torch.zeros(4, 2), torch.zeros(4, 2), torch.zeros(3, 2, 2), _groups())
    with pytest.raises(ValueError, match="g: must be on a CUDA device"):
        gm.orthogonalize(torch.zeros(3, 4))


def test_group_rows_arguments(host_checks):
    with pytest.raises(TypeError):
        gm.group_rows([0, 1], 2)
    with pytest.raises(ValueError, match="dtype"):
        gm.group_rows(torch.zeros(4), 3)
    with pytest.raises(ValueError, match="shape"):
        gm.group_rows(torch.zeros(2, 2, 2, dtype=torch.int64), 3)
    with pytest.raises(ValueError, match="positive"):
        gm.group_rows(torch.zeros(4, dtype=torch.int64), 0)
    with pytest.raises(ValueError, match="choice"):
        gm.group_rows(torch.zeros(4, 0, dtype=torch.int64), 3)
    with pytest.raises(nat.UnsupportedShape, match="routing window"):
        gm.group_rows(torch.zeros(4, dtype=torch.int64), 16385)


def test_product_arguments(host_checks):
    x, w, groups = torch.zeros(4, 2), torch.zeros(3, 2, 5), _groups()
    with pytest.raises(TypeError, match="RowGroups"):
        gm.grouped_matmul(x, w, (1, 2))
    with pytest.raises(ValueError, match="weight must have shape"):
        gm.grouped_matmul(x, torch.zeros(2, 2, 5), groups)
    with pytest.raises(ValueError, match="not be empty"):
        gm.grouped_matmul(x, torch.zeros(3, 0, 5), groups)
    with pytest.raises(ValueError, match="x must have shape"):
        gm.grouped_matmul(torch.zeros(5, 2), w, groups)
    with pytest.raises(ValueError, match="dtype"):
        gm.grouped_matmul(x.half(), w, groups)
    with pytest.raises(TypeError, match="not supported"):
        gm.grouped_matmul(x.double(), w.double(), groups)
    with pytest.raises(ValueError, match="bias must have shape"):
        gm.grouped_matmul(x, w, groups, bias=torch.zeros(5))
    with pytest.raises(ValueError, match="grad_out must have shape"):
        gm.grouped_matmul_backward(torch.zeros(4, 2), x, w, groups)
    with pytest.raises(ValueError, match="requires grad"):
        gm.grouped_matmul(x.clone().requires_grad_(), w, groups)
    short = groups._replace(order=groups.order[:3])
    with pytest.raises(ValueError, match="groups"):
        gm.grouped_matmul(x, w, short)
    with pytest.raises(ValueError, match="groups"):
        gm.grouped_matmul(x, w, groups._replace(tiles=groups.tiles[:-1]))
    with pytest.raises(ValueError, match="groups"):
        gm.grouped_matmul(x, w, groups._replace(offsets=groups.offsets.long()))


def test_orthogonalize_arguments(host_checks):
    g = torch.zeros(3, 4)
    for bad, match in ((dict(steps=-1), "steps"), (dict(steps=101), "steps"), (dict(coefficients=(1.0, 2.0)), "three"),
                       (dict(coefficients=(1.0, float("nan"), 0.0)), "finite"), (dict(eps=-1.0), "eps"),
                       (dict(eps=float("inf")), "eps"), (dict(coefficients=(4.0, 0.0, 0.0)), "diverge")):
        with pytest.raises(ValueError, match=match):
            gm.orthogonalize(g, **bad)
    with pytest.raises(ValueError, match="shape"):
        gm.orthogonalize(torch.zeros(3))
    with pytest.raises(ValueError, match="shape"):
        gm.orthogonalize(torch.zeros(3, 0))
    experts._check_polynomial(*experts.NEWTON_SCHULZ, 100)
    experts._check_polynomial(1.5, -0.5, 0.0, 100)
    experts._check_polynomial(2.0, -1.5, 0.5, 100)


def test_c_abi_refuses_before_any_cuda_call():
    lib = nat.load()
    buf = ctypes.create_string_buffer(1024 + 256)
    ws = (ctypes.addressof(buf) + 255) // 256 * 256
    one = ctypes.addressof(buf)
    assert lib.gmmxx_group_tiles_len(1 << 31, 4) == -1 and b"32-bit" in lib.gmmxx_last_error()
    assert lib.gmmxx_group_rows_workspace_bytes(-1, 4) == 0
    assert lib.gmmxx_group_rows(one, 2, 4, 3, one, one, one, ws, 1024, None) == nat.ERR_INVALID
    assert lib.gmmxx_group_rows(None, 4, 4, 3, one, one, one, ws, 1024, None) == nat.ERR_INVALID
    assert lib.gmmxx_group_rows(one, 4, 1 << 20, 3, one, one, one, ws, 16, None) == nat.ERR_WORKSPACE
    args = (4, 1, 3, 8, 8)
    assert lib.gmmxx_grouped_matmul(9, one, *args, one, one, one, one, 0, None, one, ws, 1024, None) == nat.ERR_INVALID
    assert lib.gmmxx_grouped_matmul(0, None, *args, one, one, one, one, 0, None, one, ws, 1024, None) == nat.ERR_INVALID
    assert lib.gmmxx_grouped_matmul(0, one, *args, one, one, one, one, 0, None, one, ws + 8, 1024, None) == nat.ERR_INVALID
    assert lib.gmmxx_grouped_matmul(0, one, 4, 1, 3, 8, 1 << 21, one, one, one, one, 0, None, one, ws, 1024,
                                    None) == nat.ERR_UNSUPPORTED
    assert lib.gmmxx_grouped_matmul_backward(0, None, one, *args, one, one, one, one, 0, one, None, None, ws, 1024,
                                             None) == nat.ERR_INVALID
    assert lib.gmmxx_grouped_matmul_backward(0, one, one, *args, one, one, one, one, 0, None, None, None, None, 0,
                                             None) == nat.OK  # nothing asked for
    assert lib.gmmxx_orthogonalize(0, one, 1, 4, 4, 101, 1.0, 0.0, 0.0, 0.0, one, ws, 1024, None) == nat.ERR_INVALID
    assert lib.gmmxx_orthogonalize(0, one, 1, 1 << 17, 4, 5, 1.0, 0.0, 0.0, 0.0, one, ws, 1024,
                                   None) == nat.ERR_UNSUPPORTED
    assert lib.gmmxx_orthogonalize(0, one, 1, 4, 4, 5, float("nan"), 0.0, 0.0, 0.0, one, ws, 1024,
                                   None) == nat.ERR_INVALID
