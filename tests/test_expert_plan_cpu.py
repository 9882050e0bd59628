"""CPU tier: the plan of a grouped product (expert_plan.h, built here for the host) -- which sizes run which way, so that a rule that
moves cannot silently take a way's tests along, and that every tile stays within the 31 bits its byte offsets have."""
import ctypes
import subprocess

import pytest

from tests.expert_shapes import COARSE, FEW, MX4, SEVERAL, WEIGHT

SOURCE = """
#include "expert_plan.h"
extern "C" int plan_of(const sm3_expert_desc* d, int mx4, long* out) {
  const int rc = sm3x::check_desc(d, mx4 != 0);
  if (rc) return rc;
  const sm3x::Plan p = sm3x::make_plan(d, mx4 != 0);
  const long v[] = {p.bm, p.bn, p.coarse, p.splits, p.units, p.per_xcd, p.part_bytes != 0, p.p_bytes != 0, p.q_bytes != 0};
  for (int i = 0; i < 9; i++) out[i] = v[i];
  return sm3x::fits(p) ? 0 : SM3_ERR_UNSUPPORTED;
}
"""
NT, NN, TN = range(3)


@pytest.fixture(scope='module')
def plan(tmp_path_factory):
    from sm3det_amd import build
    from sm3det_amd._lib_backbone import ExpertDesc
    import os
    d = tmp_path_factory.mktemp('plan')
    (d / 'plan.hip').write_text(SOURCE)
    subprocess.run([build._hipcc(), '--offload-arch=' + build.ARCH, '--offload-host-only', '-O1', '-std=c++17', '-fPIC', '-shared',
                    '-I' + build.CSRC, '-I' + os.path.join(os.path.dirname(build.HERE), 'include'), str(d / 'plan.hip'), '-o',
                    str(d / 'plan.so')], check=True)
    f = ctypes.CDLL(str(d / 'plan.so')).plan_of
    names = ('bm', 'bn', 'coarse', 'splits', 'units', 'per_xcd', 'parts', 'copies_p', 'copies_q')

    def ask(mode, rows, experts, n, k, mx4=False, grouped=True, **kw):
        """the product `mode` of a linear layer n x k over `rows` rows"""
        red, cols = {NT: (k, n), NN: (n, k), TN: (1, k)}[mode]
        base = dict(mode=mode, type=2, out_type=2, num_groups=experts, red=red, cols=cols, rows_out=n if mode == TN else 0, rows=rows,
                    ldp=k if mode == NT else n, ldq=k, p=1 << 20, q=1 << 20, out=1 << 20, offsets=1 << 20 if grouped else None)
        if mx4:
            base.update(q_scales=1 << 20)
        desc = ExpertDesc()
        for name, v in {**base, **kw}.items():
            setattr(desc, name, v)
        out = (ctypes.c_long * 9)()
        rc = f(ctypes.byref(desc), int(mx4), out)
        return dict(zip(names, out)) if rc == 0 else rc
    return ask


def _row_tiles(rows, offsets, bm):
    tiles = [(b - a + bm - 1) // bm for a, b in zip([0] + offsets, offsets + [rows])]
    return sum(tiles)


@pytest.mark.parametrize('name', COARSE)
def test_the_large_tiles_sizes(plan, name):
    rows, offsets, n, k, coarse, left = COARSE[name]
    for mode, want in zip((NT, NN), coarse):
        p = plan(mode, rows, len(offsets) - 1, n, k)
        assert (p['bm'], p['bn'], p['coarse']) == ((256, 256, 1) if want else (128, 128, 0)), (name, mode)
        if want and left is not None:
            assert _row_tiles(rows, offsets, 256) * ((n if mode == NT else k) // 256) % 256 == left


def _per_workgroup(tiles, per_cu):
    return tiles / (256 * per_cu)


@pytest.mark.parametrize('name', SEVERAL)
def test_the_several_tiles_sizes(plan, name):
    rows, offsets, n, k, least = SEVERAL[name]
    for mode, want in zip((NT, NN), least):
        p = plan(mode, rows, len(offsets) - 1, n, k)
        cols = n if mode == NT else k
        assert not p['coarse'] and p['splits'] == 1 and not p['copies_p'] and not p['copies_q']
        assert p['bm'] == (32 if 'of_32' in name else 128) and cols % 8 == 0
        if want > 1:
            assert _per_workgroup(_row_tiles(rows, offsets, p['bm']) * ((cols + 127) // 128), 3 if p['bm'] == 32 else 2) > want - 1


@pytest.mark.parametrize('name', WEIGHT)
def test_the_weight_gradients_sizes(plan, name):
    rows, offsets, n, k, whole, least = WEIGHT[name]
    p = plan(TN, rows, len(offsets) - 1, n, k)
    assert (p['units'] == len(offsets) - 1 and not p['parts']) == whole
    assert _per_workgroup(p['per_xcd'] * 8, 2) > least - 1


@pytest.mark.parametrize('name', MX4)
def test_the_4_bit_sizes(plan, name):
    rows, offsets, n, k, least, slices = MX4[name]
    p = plan(NT, rows, len(offsets) - 1 if offsets else 1, n, k, mx4=True, grouped=offsets is not None)
    assert p['splits'] == slices and bool(p['parts']) == (slices > 1) and n % 4 == 0
    if least > 1:
        tiles = _row_tiles(rows, offsets or [0, rows], p['bm']) * ((n + 127) // 128)
        assert _per_workgroup(tiles, 3 if p['bm'] == 32 else 2) > least - 1


@pytest.mark.parametrize('red', (1 << 12, (1 << 22) - 64, (1 << 22) - 8, (1 << 22) - 7, (1 << 22) - 1, 1 << 22))
@pytest.mark.parametrize('ld', (0, 1 << 22))
def test_the_bytes_of_a_tiles_rows_stay_below_2_to_the_31(plan, red, ld):
    """rows of the reduction's length, padded to 8 where the kernel copies them; a part of a wider matrix where ld says so"""
    for mode in (NT, NN):
        for rows in (1, 300, 4096, 70000):
            n, k = (4096, red) if mode == NT else (red, 4096)
            kw = dict(ldp=ld) if ld else {}
            if ld and mode == NT:
                kw.update(ldq=ld)
            p = plan(mode, rows, 1, n, k, **kw)
            row = (red + 7) // 8 * 8
            pitch = max(ld, row) if not p['copies_p'] else row
            assert ((p['bm'] - 1) * pitch + row) * 2 < 1 << 31, (mode, rows, p)
            assert mode == NN or ((p['bn'] - 1) * pitch + row) * 2 < 1 << 31, (mode, rows, p)
            if rows >= 4096 and red < (1 << 22) - 7:
                assert p['coarse']


def test_longer_reductions_are_refused(plan):
    for mode, n, k in ((NT, 4096, (1 << 22) + 1), (NN, (1 << 22) + 1, 4096), (TN, 4096, (1 << 22) + 1), (TN, (1 << 22) + 1, 4096)):
        assert plan(mode, 4096, 1, n, k) == -4


@pytest.mark.parametrize('name', FEW)
def test_few_rows_run_in_one_launch_while_that_is_the_faster_way(name):
    """(one launch: no workspace) -- by the rows, the experts and the sizes of the product, not by the mean load alone"""
    from sm3det_amd import _lib
    from sm3det_amd._lib_backbone import EXPERT_DESC
    rows, offsets, n, k, bf16, fp32 = FEW[name]
    a = 1 << 20
    for dtype, one in ((0, fp32), (1, bf16), (2, bf16)):
        desc = EXPERT_DESC.pack(0, dtype, dtype, 0, 0, len(offsets) - 1, k, n, 0, 0, rows, k, 0, a, a, 0, a, a, 0, 0, a)
        assert (_lib.lib().sm3_mx4_gemm_workspace_bytes(desc) == 0) == one, dtype
