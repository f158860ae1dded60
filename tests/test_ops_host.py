"""Matrix and routing entry points without a GPU: the size checks, workspace sizes and refusals that need no device,
and the tests' own 64-bit row decoder against the oracle's."""
import numpy as np
import pytest

import fronk_b200 as fb
from tests import quant


def test_matrix_check(built):
    ok = [(fb.Q4_K, 1, 256), (fb.Q4_K, 513, 2048), (fb.Q4_K, 1 << 24, 65536), (fb.MXFP4, 1, 32), (fb.MXFP4, 7, 672)]
    for a in ok:
        assert fb.matrix_check(*a) == fb.OK, a
    bad = [(fb.Q4_K, 0, 256), (fb.Q4_K, 1, 0), (fb.Q4_K, 1, 128), (fb.Q4_K, 1, 65536 + 256), (fb.MXFP4, 1, 16),
           (fb.MXFP4, (1 << 24) + 1, 32), (0, 1, 256), (13, 1, 256)]
    for a in bad:
        assert fb.matrix_check(*a) == fb.INVALID, a
    assert fb.matrix_check(fb.Q8_0, 1, 256) == fb.UNSUPPORTED


def test_routing_check(built):
    for a in [(1, 10, 10), (1, 512, 512), (1 << 24, 512, 1 << 20), (5, 512, 513, fb.BF16, fb.ROUTE_SHARED)]:
        assert fb.routing_check(*a) == fb.OK, a
    for a in [(0, 512, 512), ((1 << 24) + 1, 512, 512), (1, 9, 9), (1, 513, 513), (1, 512, 511), (1, 512, 512, 2),
              (1, 512, 512, fb.F32, fb.ROUTE_SHARED), (1, 512, 600, fb.F32, 2)]:
        assert fb.routing_check(*a) == fb.INVALID, a


def test_workspace(built):
    assert fb.balance_workspace(1, 10) > 0
    # grows with the rows up to a bound that does not depend on them
    sizes = [fb.balance_workspace(t, 512) for t in (1, 100, 10000, 1 << 20, 1 << 24)]
    assert sizes == sorted(sizes) and sizes[-1] == sizes[-2] <= 4 << 20
    for t, e in [(0, 512), (1, 9), (1, 513), ((1 << 24) + 1, 64)]:
        with pytest.raises(fb.FrcError):
            fb.balance_workspace(t, e)


def test_null_context_is_refused(built):
    lib = fb.library()
    assert lib.frc_matrix_open(None, fb.Q4_K, 1, 256, None, 144, None) == fb.INVALID
    assert lib.frc_matrix_close(None) == fb.INVALID
    assert lib.frc_matvec_device(None, None, 1, None, 0, 0, None, 0, 0, None) == fb.INVALID
    assert lib.frc_route_device(None, 1, 512, None, 512, 0, None, None, None, 0, None, None) == fb.INVALID
    assert lib.frc_balance_device(None, 1, 512, None, 512, 0, None, None, None, None) == fb.INVALID
    assert lib.frc_route_backward_device(None, 1, 512, None, 512, 0, None, None, None, None, None, None, 512, 0,
                                         None) == fb.INVALID


@pytest.mark.parametrize("type_,n", [(fb.Q4_K, 512), (fb.MXFP4, 96)])
def test_decoder_against_oracle(built, oracle, type_, n):
    rng = np.random.default_rng(5)
    raw = quant.random_rows(type_, 8, n, rng, exponents=(0, 254))
    w, _ = quant.weights(type_, raw, n)
    for r in range(8):
        rc, ref = oracle.decode_row(raw[r], type_, n)
        assert rc == fb.OK
        # the oracle narrows each weight to fp32 once: half a step of the terms it is the difference of
        assert np.all(np.abs(ref - w[r]) <= 2.0 ** -23 * np.abs(quant.weights(type_, raw[r:r + 1], n)[1][0]) + 2.0 ** -149)
