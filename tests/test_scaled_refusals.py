"""Argument checks of block quantisation, block-scaled contraction and cross entropy. They are made before any device work,
so they run without a GPU, on a handle whose memory is zeros."""
import ctypes

import pytest

import hiptensor_b200 as ht
from hiptensor_b200 import _lib

INVALID, UNSUPPORTED = ht.STATUS_INVALID_VALUE, ht.STATUS_NOT_SUPPORTED
E4, E5, BF, F32, F64 = ht.R_8F_E4M3, ht.R_8F_E5M2, ht.R_16BF, ht.R_32F, ht.R_64F


class HostHandle(ht.Handle):
    def __init__(self):
        from hiptensor_b200 import build

        build.build()
        self._L = _lib.lib()
        self._mem = ctypes.create_string_buffer(1 << 16)
        self._h = ctypes.c_void_p(ctypes.addressof(self._mem))

    def destroy(self):
        self._h = None


@pytest.fixture(scope="module")
def h():
    return HostHandle()


def packed(lens):
    s, out = 1, []
    for n in reversed(lens):
        out.append(s)
        s *= max(n, 1)
    return out[::-1]


def desc(h, lens, kind, strides=None):
    return h.tensor_descriptor(lens, strides or packed(lens), kind)


def quantize_status(h, lens=(200, 300), modeA=(0, 1), block=(1, 128), typeA=BF, lensQ=None, modeQ=None, typeQ=E4, lensS=None,
                    typeS=F32, stridesQ=None):
    lensQ = lens if lensQ is None else lensQ
    modeQ = modeA if modeQ is None else modeQ
    lensS = [-(-n // b) for n, b in zip(lens, block)] if lensS is None else lensS
    try:
        h.block_quantize(0, desc(h, lens, typeA), modeA, block, 0, desc(h, lensQ, typeQ, stridesQ), modeQ, 0, desc(h, lensS, typeS))
    except ht.HiptensorError as e:
        return e.status
    return 0


@pytest.mark.parametrize("want,kw", [
    (ht.STATUS_NOT_INITIALIZED, {}),  # good arguments: only the handle has no device
    (ht.STATUS_NOT_INITIALIZED, dict(block=(128, 128), typeA=F32, typeQ=E5)),
    (ht.STATUS_NOT_INITIALIZED, dict(lens=(3, 200, 300), modeA=(5, 0, 1), block=(1, 128, 128))),
    (ht.STATUS_NOT_INITIALIZED, dict(lensQ=(300, 200), modeQ=(1, 0))),
    (UNSUPPORTED, dict(typeA=F64)), (UNSUPPORTED, dict(typeA=E4)), (UNSUPPORTED, dict(typeQ=BF)), (INVALID, dict(typeS=F64)),
    (INVALID, dict(block=(1, 1))), (INVALID, dict(block=(1, 64), lensS=(200, 5))), (INVALID, dict(block=(0, 128), lensS=(200, 3))),
    (INVALID, dict(lensS=(200, 2))), (INVALID, dict(lensS=(200, 4))), (INVALID, dict(lensQ=(200, 299))),
    (INVALID, dict(modeQ=(0, 2))), (INVALID, dict(modeA=(1, 1), modeQ=(1, 1))), (INVALID, dict(stridesQ=(0, 1))),
    (UNSUPPORTED, dict(lens=(300, 300, 300), modeA=(0, 1, 2), block=(128, 128, 128))),
])
def test_quantize(h, want, kw):
    assert quantize_status(h, **kw) == want


def test_quantize_lists_have_the_descriptors_rank(h):
    assert quantize_status(h, modeA=(0,), modeQ=(0, 1), block=(1, 128), lensS=(200, 3)) == INVALID
    assert quantize_status(h, block=(128,), lensS=(2, 3)) == INVALID


def scaled_status(h, m=200, n=300, k=400, blockA=(1, 128), blockB=(128, 128), tA=E4, tB=E5, tD=BF, modeA=(0, 2), modeB=(1, 2),
                  modeD=(0, 1), lensA=None, lensB=None, lensD=None, c=None, sA=None, compute=ht.COMPUTE_32F):
    lensA, lensB, lensD = lensA or (m, k), lensB or (n, k), lensD or (m, n)
    ceil = lambda lens, b: [-(-x // y) for x, y in zip(lens, b)]  # noqa: E731
    try:
        h.scaled_contraction_plan(desc(h, lensA, tA), modeA, desc(h, sA or ceil(lensA, blockA), F32), blockA, desc(h, lensB, tB),
                                  modeB, desc(h, ceil(lensB, blockB), F32), blockB, c(h) if c else None, desc(h, lensD, tD), modeD,
                                  compute)
    except ht.HiptensorError as e:
        return e.status
    return 0


@pytest.mark.parametrize("want,kw", [
    (0, {}), (0, dict(m=1, n=1, k=1)), (0, dict(m=0)), (0, dict(k=0)), (0, dict(tD=F32)), (0, dict(modeD=(1, 0), lensD=(300, 200))),
    (0, dict(lensA=(4, 50, 400), modeA=(3, 4, 2), blockA=(1, 1, 128), lensD=(4, 50, 300), modeD=(3, 4, 1))),
    (0, dict(c=lambda h: desc(h, (200, 300), BF))),
    (UNSUPPORTED, dict(c=lambda h: desc(h, (200, 300), F32))), (UNSUPPORTED, dict(c=lambda h: desc(h, (200, 300), BF, (1, 200)))),
    (UNSUPPORTED, dict(tA=BF)), (UNSUPPORTED, dict(tD=E4)), (UNSUPPORTED, dict(tD=F64)), (UNSUPPORTED, dict(compute=ht.COMPUTE_16F)),
    (UNSUPPORTED, dict(blockA=(1, 1))), (UNSUPPORTED, dict(blockB=(128, 1))), (INVALID, dict(blockA=(64, 128), sA=(4, 4))),
    (INVALID, dict(sA=(200, 3))), (INVALID, dict(lensB=(300, 401))), (INVALID, dict(lensD=(200, 301))), (INVALID, dict(modeD=(0, 0))),
    (INVALID, dict(modeA=(0, 3))), (INVALID, dict(modeD=(0, 7))), (INVALID, dict(lensA=(200, 400), modeA=(0, 2), lensD=(300,), modeD=(1,))),
    # a batch mode, two contracted modes, free modes that do not fold
    (UNSUPPORTED, dict(lensA=(9, 200, 400), modeA=(9, 0, 2), blockA=(1, 1, 128), lensB=(9, 300, 400), modeB=(9, 1, 2),
                       blockB=(1, 128, 128), lensD=(9, 200, 300), modeD=(9, 0, 1))),
    (UNSUPPORTED, dict(lensA=(200, 4, 400), modeA=(0, 3, 2), blockA=(1, 128, 128), lensB=(300, 4, 400), modeB=(1, 3, 2),
                       blockB=(128, 128, 128))),
    (UNSUPPORTED, dict(lensA=(4, 50, 400), modeA=(3, 4, 2), blockA=(1, 1, 128), lensD=(50, 4, 300), modeD=(4, 3, 1))),
])
def test_scaled(h, want, kw):
    assert scaled_status(h, **kw) == want


def ce_status(h, lensH=(100, 64), modeH=(0, 2), lensW=(1000, 64), modeW=(1, 2), t=BF, tW=None, sH=None, sW=None,
              compute=ht.COMPUTE_32F):
    try:
        h.cross_entropy_plan(desc(h, lensH, t, sH), modeH, desc(h, lensW, t if tW is None else tW, sW), modeW, -100, compute)
    except ht.HiptensorError as e:
        return e.status
    return 0


@pytest.mark.parametrize("want,kw", [
    (0, {}), (0, dict(t=F32)), (0, dict(lensH=(0, 64))), (0, dict(lensH=(1, 1), lensW=(1, 1))),
    (0, dict(lensH=(4, 9, 64), modeH=(5, 0, 2), sH=(640, 64, 1))), (0, dict(lensW=(64, 1000), modeW=(2, 1))),
    (UNSUPPORTED, dict(t=F64)), (UNSUPPORTED, dict(t=E4)), (UNSUPPORTED, dict(tW=F32)), (UNSUPPORTED, dict(compute=ht.COMPUTE_16F)),
    (INVALID, dict(lensW=(0, 64))), (INVALID, dict(lensH=(100, 0), lensW=(1000, 0))), (INVALID, dict(lensH=(100, 63))),
    (INVALID, dict(modeH=(0, 3))), (INVALID, dict(modeH=(2, 2))), (INVALID, dict(modeW=(2, 2))), (INVALID, dict(sH=(64, 0))),
    (UNSUPPORTED, dict(lensW=(10, 100, 64), modeW=(3, 1, 2), sW=(12800, 64, 1))),
    (UNSUPPORTED, dict(lensH=(100, 8, 8), modeH=(0, 2, 3), lensW=(1000, 8, 8), modeW=(1, 2, 3), sW=(640, 80, 1))),
])
def test_cross_entropy(h, want, kw):
    assert ce_status(h, **kw) == want


def test_cross_entropy_workspace(h):
    plan = h.cross_entropy_plan(desc(h, (1000, 64), BF), (0, 2), desc(h, (32001, 64), BF), (1, 2))
    for gradient in (False, True):
        least, some, most = [h.cross_entropy_workspace_size(plan, gradient, p)
                             for p in (ht.WORKSPACE_MIN, ht.WORKSPACE_RECOMMENDED, ht.WORKSPACE_MAX)]
        assert 0 < least <= some <= most
    with pytest.raises(ht.HiptensorError):
        h.cross_entropy_workspace_size(plan, False, 9)
    none = h.cross_entropy_plan(desc(h, (0, 64), BF), (0, 2), desc(h, (32001, 64), BF), (1, 2))
    assert h.cross_entropy_workspace_size(none, True) == 0


@pytest.mark.parametrize("t,status", [((1 << 31) // 3 - 300, 0), ((1 << 31) // 3 - 100, UNSUPPORTED), (1 << 30, UNSUPPORTED)])
def test_cross_entropy_of_more_f32_tokens_than_three_parts_can_be_counted(h, t, status):
    """Coordinates of loads are 32-bit numbers, and the three parts of f32 tokens follow each other."""
    assert ce_status(h, lensH=(t, 1), lensW=(1000, 1), t=F32) == status
    assert ce_status(h, lensH=(t, 1), lensW=(1000, 1), t=BF) == 0


@pytest.mark.parametrize("gradient,times", [(False, 3), (True, 6)])
def test_cross_entropy_pieces_of_f32_stay_countable(h, gradient, times):
    """The largest workspace holds the parts of a piece of at most 2^31 / 3 (gradient: / 6) classes, 8 elements a row here."""
    v = (1 << 30) + 12345
    plan = h.cross_entropy_plan(desc(h, (20, 8), F32), (0, 2), desc(h, (v, 8), F32), (1, 2))
    most = h.cross_entropy_workspace_size(plan, gradient, ht.WORKSPACE_MAX)
    per_class = 3 * 8 * 2 + (3 * 64 * 2 if gradient else 20 * 8 / 128)
    assert most >= (1 << 31) / times * 0.99 * per_class
    assert most <= (1 << 31) / times * per_class + (1 << 20)


def test_null_arguments(h):
    L = _lib.lib()
    p = ctypes.c_void_p(0)
    assert L.htBlockQuantize(None, None, None, None, None, None, None, None, None, None, None) == 1
    assert L.htCreateScaledContractionPlan(h._h, ctypes.byref(p), *([None] * 11), 4) == 1
    assert L.htCreateCrossEntropyPlan(h._h, ctypes.byref(p), None, None, None, None, 0, 4) == 1
    assert L.htScaledContraction(h._h, *([None] * 10)) == 1
    assert L.htCrossEntropy(h._h, *([None] * 8), 0, None) == 1
    assert L.htCrossEntropyGradient(h._h, *([None] * 10), 0, None) == 1
    assert L.htCrossEntropyGetWorkspaceSize(h._h, None, 0, 2, None) == 1
    assert L.htDestroyScaledContractionPlan(None) == 0 and L.htDestroyCrossEntropyPlan(None) == 0


def test_eight_bit_tensors_stay_out_of_the_other_operations(h):
    d = desc(h, (16, 16), E4)
    c = h.contraction_descriptor(d, (0, 2), d, (1, 2), None, None, desc(h, (16, 16), F32), (0, 1), ht.COMPUTE_32F)
    assert c is not None  # as for every descriptor, the types are looked at when a plan is made
    with pytest.raises(ht.HiptensorError) as e:
        ht.describe_contraction_plan((16, 16), (16, 1), (0, 2), E4, (16, 16), (16, 1), (1, 2), E4, (16, 16), (16, 1), (0, 1), F32,
                                     False, ht.COMPUTE_32F)
    assert e.value.status == UNSUPPORTED
    with pytest.raises(ht.HiptensorError):
        ht.describe_permutation_plan((16, 16), (0, 1), (1, 0), E4)
