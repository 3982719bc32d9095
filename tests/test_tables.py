"""Constant tables: generated by nnsp_amd/tables.py from closed-form rules and
checked word-for-word against the reference's source tables."""
import os
import re

import numpy as np
import pytest

from conftest import REFERENCE, ROOT, needs_reference
from nnsp_amd import tables


def test_generated_files_up_to_date():
    with open(os.path.join(ROOT, "nnsp_amd", "csrc", "gen", "nnsp_tables.h")) as f:
        assert f.read() == tables.header_text()
    with open(os.path.join(ROOT, "nnsp_amd", "csrc", "gen", "nnsp_tables_export.c")) as f:
        assert f.read() == tables.export_text()


def _c_table(path, name):
    text = open(path, encoding="utf-8-sig").read()
    m = re.search(re.escape(name) + r"\s*\[\s*\]\s*=\s*\{([^}]*)\}", text)
    vals = [int(v, 16) for v in re.findall(r"0x[0-9a-fA-F]+", m.group(1))]
    return np.array([v - 65536 if v >= 32768 else v for v in vals])


@needs_reference
@pytest.mark.parametrize("fname,sym,gen", [
    ("window_stft_coef.c", "stft_win_coeff", tables.stft_window),
    ("melSpec_coeff.c", "mfltrBank_coeff", tables.mel_bank_packed),
    ("fixlog10.c", "log_tayler_coeff", tables.log_interp),
    ("activation.c", "coeffs_tanh", tables.tanh_interp),
])
def test_source_tables_exact(fname, sym, gen):
    ref = _c_table(os.path.join(REFERENCE, "ns-nnsp", "src", fname), sym)
    np.testing.assert_array_equal(gen().astype(np.int64), ref)


def test_mel_segments_per_bank_fit_fe_kernel():
    """fe_kernel sums each Mel bank over at most FE_MEL_MAXSEG lane segments
    (unrolled, nnsp_kernels.hip); the generated segment table must fit that."""
    src = open(os.path.join(ROOT, "nnsp_amd", "csrc", "kernels", "nnsp_kernels.hip")).read()
    maxseg = int(re.search(r"#define FE_MEL_MAXSEG (\d+)", src).group(1))
    seg = tables.mel_segments().reshape(-1, 4)
    banks = seg[:, 0]
    counts = np.bincount(banks[banks < 40], minlength=40)
    assert counts.min() >= 1 and counts.max() <= maxseg
    # a bank's segments are consecutive lanes, and lane 63 has none: fe_kernel
    # reads its (zero) partial sum for a bank's missing segments
    for b in range(40):
        lanes = np.nonzero(banks == b)[0]
        assert (np.diff(lanes) == 1).all()
    assert seg[63, 2] == 0 and banks[63] >= 40
    # each lane reads FE_MEL_LEN power-spectrum bins from its segment start
    # (zero coefficients past the segment's own): they must stay inside FE_P_DW
    pdw = int(re.search(r"#define FE_P_DW (\d+)", src).group(1))
    mlen = int(re.search(r"#define FE_MEL_LEN (\d+)", src).group(1))
    assert seg[:, 1].max() + mlen <= pdw and seg[:, 2].max() <= mlen


@needs_reference
def test_portable_fft_tables_exact():
    """twiddle_fft_dif.c (ARM_OPTIMIZED=0): fft_tw_coeff / rfft_tw_coeff
    (COMPLEX16 words) and br_coeff, word for word (row N4)."""
    text = open(os.path.join(REFERENCE, "ns-nnsp", "src", "twiddle_fft_dif.c"), encoding="utf-8-sig").read()

    def words(name):
        m = re.search(re.escape(name) + r"\s*\[\s*\]\s*=\s*\{([^}]*)\}", text)
        v = np.array([int(x, 0) for x in re.findall(r"0x[0-9a-fA-F]+|\d+", m.group(1))], np.int64)
        return np.where(v >= 2 ** 31, v - 2 ** 32, v)

    np.testing.assert_array_equal(tables.dif_twiddles().astype(np.int64), words("fft_tw_coeff"))
    np.testing.assert_array_equal(tables.rfft_dif_twiddles().astype(np.int64), words("rfft_tw_coeff"))
    np.testing.assert_array_equal(tables.bitrev8().astype(np.int64), words("br_coeff"))


def test_fft_tables_are_the_nearest_q31_values():
    """Twiddles and split coefficients are cos and sin to the nearest q31
    value, half a step off at most (1 itself, which q31 has not, saturates);
    cos and sin here from their series in exact fractions."""
    from fractions import Fraction

    pi = Fraction(31415926535897932384626433832795028841971693993751, 10 ** 49)

    def sin(n, d):  # of 2 pi n / d
        x, t, out = 2 * pi * n / d, Fraction(1), Fraction(0)
        if 4 * n > d:  # to the first quadrant
            return sin(d - n, d) * -1 if 2 * n > d else sin(d - 2 * n, 2 * d)
        t = x = Fraction(x).limit_denominator(10 ** 30)
        for k in range(1, 16):
            out += t
            t = Fraction(-t * x * x / ((2 * k) * (2 * k + 1))).limit_denominator(10 ** 30)
        return out

    def cos(n, d):
        return sin((4 * n + d) % (4 * d), 4 * d)

    def check(got, value):
        # cos and sin of the generator are doubles: 2^31 times half a unit in their last place beyond the half step
        exact = min(value * 2 ** 31, 2 ** 31 - 1)
        assert abs(int(got) - exact) <= Fraction(1, 2) + Fraction(1, 10 ** 6)

    tw = tables.cfft256_twiddles().reshape(-1, 2)
    for i in range(192):
        check(tw[i, 0], 1 if i == 0 else cos(i, 256))
        check(tw[i, 1], sin(i, 256))
    split = tables.rfft512_split_coefs().reshape(-1, 3)
    for k in range(256):
        s, c = sin(k, 512), 1 if k == 0 else cos(k, 512)
        check(split[k, 0], (1 - s) / 2)
        check(split[k, 1], -Fraction(c) / 2)
        check(split[k, 2], (1 + s) / 2)


def test_split_coefficients_are_symmetric():
    """fe_kernel splits bins k and 256 - k together (nnsp_dev.h split_pair),
    which relies on realCoefA/B at 16k being symmetric: A1[256-k] = A1[k],
    A2[256-k] = -A2[k], B1[256-k] = B1[k]."""
    from nnsp_amd import tables
    c = np.asarray(tables.rfft512_split_coefs(), np.int64).reshape(256, 3)
    k = np.arange(1, 256)
    np.testing.assert_array_equal(c[256 - k, 0], c[k, 0])
    np.testing.assert_array_equal(c[256 - k, 1], -c[k, 1])
    np.testing.assert_array_equal(c[256 - k, 2], c[k, 2])


def test_tanh_shifted_table_matches_activation_c():
    """tanh_q15s (nnsp_dev.h: the split NN kernels' lookup on nnsp_tbl_tanh1)
    equals activation.c's tanh (the oracle's restatement, pinned to the
    reference by test_oracle_pinned) for every |x| < 2^18 and far beyond."""
    t = tables.tanh_interp().astype(np.int64).reshape(-1, 2)
    t1 = tables.tanh_interp_shifted().astype(np.int64).reshape(-1, 2)
    assert t1.shape == (256, 2)
    x = np.concatenate([np.arange(-(1 << 18), 1 << 18, dtype=np.int64),
                        np.array([2**31 - 1, -(2**31 - 1), 2**30, -2**30, 196607, 196608, 262143 * 1000])])
    # activation.c:31-69 (as nnsp_dev.h tanh_q15)
    a = np.abs(x)
    kx = np.clip((a - 512) >> 10, 0, 191)
    dx = (a - 512) - (kx << 10)
    v = t[kx, 0] + ((dx * t[kx, 1]) >> 15)
    y = np.where(a >= 5 << 15, 0x7FFF, np.maximum(v, 0))
    ref = np.where(x < 0, -y, y)
    # tanh_q15s: index (|x| + 512) >> 10 (8 bits), offset (|x| + 512) & 1023
    bb = a + 512
    k1 = (bb >> 10) & 255
    v1 = t1[k1, 0] + (((bb & 1023) * t1[k1, 1]) >> 15)
    y1 = np.where(a >= 5 << 15, 0x7FFF, np.maximum(v1, 0))
    s = np.where(x < 0, -1, 0)
    got = (y1 ^ s) - s
    np.testing.assert_array_equal(got, ref)


def _act_affine(x, fn):
    """nnsp_dev.h act_q15<fn> in numpy (uint32 / int32 wraps as on the GPU)."""
    tb = tables.act_affine_table().astype(np.int64)
    x = x.astype(np.int64)
    sgn = (x < 0).astype(np.int64)
    s = -sgn
    bb = (((x ^ s) & 0xFFFFFFFF) + 512 + sgn) & 0xFFFFFFFF
    bb = np.minimum(bb, 164352)
    dx = bb & 511
    k = ((bb >> 5) & 0x1FF0) >> 4
    A = tb[k, 2 * sgn]
    b = tb[k, 2 * sgn + 1]
    z = (A + dx * b) & 0xFFFFFFFF
    if fn == 0:
        zs = np.where(z >= 1 << 31, z - (1 << 32), z)
        return zs >> 15
    return ((z + (1 << 30)) & 0xFFFFFFFF) >> 16


def test_act_affine_tables_match_activation_c():
    """act_q15 (nnsp_dev.h: one v_mad_i32_i24 on tables.act_affine_table,
    the sign and saturation folded into the tables and an index clamp) equals
    activation.c's tanh_fix (:31-69) and sigmoid_fix (:72-83) on every input
    of |x| < 2^18 and at the int32 extremes."""
    t = tables.tanh_interp().astype(np.int64).reshape(-1, 2)
    x = np.concatenate([np.arange(-(1 << 18), 1 << 18, dtype=np.int64),
                        np.array([2**31 - 1, -2**31, -(2**31 - 1), 2**30, -2**30, 163839, 163840, -163840,
                                  -163841, 164351, 164352, -164352, 262143 * 1000])])

    def tanh_ref(v):
        a = np.abs(v)
        kx = np.clip((a - 512) >> 10, 0, 191)
        dx = (a - 512) - (kx << 10)
        y = np.where(a >= 5 << 15, 0x7FFF, np.maximum(t[kx, 0] + ((dx * t[kx, 1]) >> 15), 0))
        return np.where(v < 0, -y, y)

    assert tables.act_affine_table().shape == (tables.ACT_ENTRIES, 4)
    np.testing.assert_array_equal(_act_affine(x, 0), tanh_ref(x))
    # sigmoid_fix(v) = (tanh(v >> 1) >> 1) + 16384; act_q15<1> takes w = v >> 1
    np.testing.assert_array_equal(_act_affine(x, 1), (tanh_ref(x) >> 1) + 16384)
