"""The paged-cache operators without a GPU: their index arithmetic (a host build of
csrc/paged.h), their refusals, and the C ABI's argument errors."""
import os
import shutil
import subprocess

import pytest
import torch

import paged_reference as ref
import vecattention_amd as va
from vecattention_amd import _native as nat

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "vecattention_amd", "csrc")

PROG = r"""
#include "paged.h"
#include <cstdio>
#include <cstdlib>
#include <vector>
static uint64_t rng = 88172645463325252ull;
static uint32_t rnd() { rng ^= rng << 13; rng ^= rng >> 7; rng ^= rng << 17; return uint32_t(rng >> 16); }
int main() {
  // n / d for the divisors at and beside powers of two, and any others
  std::vector<uint32_t> ds = {1, 2, 3, 5, 7, 12, 24, 48, 100, 0x7ffffffeu, 0x7fffffffu};
  for (int s = 1; s < 31; ++s)
    for (int e = -1; e < 2; ++e) ds.push_back((1u << s) + e);
  for (int i = 0; i < 2000; ++i) ds.push_back(rnd() % 0x7fffffffu + 1);
  for (uint32_t d : ds) {
    if (!d) continue;
    const va::FastDiv f(d);
    auto check = [&](uint64_t n) {
      if (n >= 0x80000000ull) return;
      if (f.div(uint32_t(n)) != n / d) { printf("BAD div %llu / %u\n", (unsigned long long)n, d); exit(1); }
    };
    for (uint64_t k = 0; k < 4; ++k)
      for (int e = -1; e < 2; ++e) {
        check(uint64_t(d) * k + e + (k == 0 && e < 0));
        check(0x7fffffffull / d * d + e - 1 + (e < 0));
      }
    for (int i = 0; i < 500; ++i) check(rnd() & 0x7fffffffu);
    check(0x7fffffffu);
  }
  // every unit has one owner, shares are in order and differ by at most one
  for (uint32_t total : {1, 2, 7, 100, 1023, 4096, 100003})
    for (uint32_t groups : {1, 2, 3, 64, 511, 512, 2048}) {
      const va::PagedShare s(total, groups);
      if (s.begin(0) != 0 || s.begin(groups) != total) { printf("BAD ends\n"); return 1; }
      for (uint32_t w = 0; w < groups; ++w) {
        const uint32_t n = s.begin(w + 1) - s.begin(w);
        if (n < total / groups || n > total / groups + 1) { printf("BAD share\n"); return 1; }
        for (uint32_t u = s.begin(w); u < s.begin(w + 1); ++u)
          if (s.owner(u) != w) { printf("BAD owner\n"); return 1; }
      }
    }
  // keys and units of a request
  if (va::paged_keys(-5, 100) != 0 || va::paged_keys(0, 0) != 0 || va::paged_keys(100, 100) != 100 ||
      va::paged_keys(101, 100) != -1 || va::paged_keys(1, 0) != -1 ||
      va::paged_keys(0x7fffffff, int64_t(1) << 40) != 0x7fffffff) { printf("BAD keys\n"); return 1; }
  if (va::paged_units(0, 128) != 1 || va::paged_units(-1, 128) != 1 || va::paged_units(128, 128) != 1 ||
      va::paged_units(129, 128) != 2 || va::paged_units(0x7fffffff, 128) != 16777216) { printf("BAD units\n"); return 1; }
  // pages and slots of a request; ids that are no pages
  const int32_t row[4] = {9, -1, 4, 7}, list[3] = {20, 21, -5};
  const va::PlanRow r(33, 30, 16, 4);
  if (r.held != 3 || r.need != 1) { printf("BAD need\n"); return 1; }
  if (va::plan_slot(r, 0, 16, 4, row, list, 3, 0) != 144 || va::plan_slot(r, 17, 16, 4, row, list, 3, 0) != -1 ||
      va::plan_slot(r, 47, 16, 4, row, list, 3, 0) != 79 || va::plan_slot(r, 48, 16, 4, row, list, 3, 1) != 336 ||
      va::plan_slot(r, 48, 16, 4, row, list, 3, 2) != -1 || va::plan_slot(r, 48, 16, 4, row, list, 3, 3) != -1 ||
      va::plan_slot(r, 48, 16, 4, row, list, 3, -1) != -1 || va::plan_slot(r, 64, 16, 4, row, list, 3, 0) != -1) {
    printf("BAD slot\n"); return 1; }
  if (va::PlanRow(-4, -2, 16, 4).need || va::PlanRow(0, 100, 16, 4).need != 4 || va::PlanRow(100, 5, 16, 4).need ||
      va::PlanRow(0x7fffffff, 0x7fffffff, 1, 0x7fffffff).need) { printf("BAD row\n"); return 1; }
  const int32_t big[1] = {0x7fffffff};
  if (va::plan_slot(va::PlanRow(5, 1, 1u << 30, 1), 5, 1u << 30, 1, big, list, 3, 0) !=
      int64_t(0x7fffffff) * (int64_t(1) << 30) + 5) { printf("BAD 64\n"); return 1; }
  printf("OK\n");
  return 0;
}
"""


def test_index_arithmetic(tmp_path):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("no hipcc")
    src = tmp_path / "paged.cpp"
    src.write_text(PROG)
    exe = tmp_path / "paged"
    subprocess.run([hipcc, "-x", "hip", "--offload-arch=gfx950", "-O2", "-std=c++17", "-I", CSRC,
                    "-o", str(exe), str(src)], check=True, capture_output=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0 and out.stdout.strip() == "OK", out.stdout + out.stderr


def test_no_matrix_result_is_read_too_soon(tmp_path):
    from asm_hazards import early_reads
    from vecattention_amd import build
    # The checker itself: a branch straight to the read is found, a wait before it is enough.
    body = ("_Zk:\n v_mfma_f32_16x16x4_f32 a[0:3], v1, v2, a[0:3]\n s_cbranch_vccnz .LBB0_1\n"
            " s_nop 15\n.LBB0_1:\n{} v_accvgpr_read_b32 v3, a3\n s_endpgm\n")
    assert len(early_reads(body.format(""))[1]) == 1
    assert early_reads(body.format(" s_nop 9\n")) == (1, [])
    out = tmp_path / "paged_attn.s"
    subprocess.run([build.hipcc(), *build.FLAGS, "--cuda-device-only", "-S",
                    os.path.join(CSRC, "paged_attn.hip"), "-o", str(out)], check=True,
                   capture_output=True)
    count, early = early_reads(out.read_text())
    assert count > 300 and early == []


def test_plain_plan_by_hand():
    table, lens, indptr, slots, pos, req, taken = ref.plan(
        [3, 0, 4], [2, 0, 5], [[8, -1, -1], [-1, -1, -1], [5, -1, -1]], [1, 2, 3], 4, 8)
    assert table == [[8, 1, -1], [-1, -1, -1], [5, 2, 3]] and taken == 3
    assert lens == [5, 0, 9] and indptr == [0, 2, 2, 7]
    assert slots == [35, 4, 8, 9, 10, 11, 12, -1]
    assert pos == [3, 4, 4, 5, 6, 7, 8, 0] and req == [0, 0, 2, 2, 2, 2, 2, -1]


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def test_plan_refusals():
    ok = dict(kv_lens=i32(3), new_lens=i32(3), block_tables=i32(3, 4), free_pages=i32(5),
              page_size=16, num_tokens=8)
    for over, err in [(dict(new_lens=i32(2)), ValueError), (dict(kv_lens=i32(3, 1)), ValueError),
                      (dict(block_tables=i32(2, 4)), ValueError),
                      (dict(free_pages=i32(5, 1)), ValueError),
                      (dict(free_head=i32(2)), ValueError),
                      (dict(kv_lens=torch.zeros(3)), TypeError),
                      (dict(free_pages=torch.zeros(5, dtype=torch.int64)), TypeError),
                      (dict(page_size=0), ValueError), (dict(num_tokens=-1), ValueError),
                      (dict(block_tables=i32(1, 4).expand(3, 4)), ValueError),
                      (dict(block_tables=i32(4, 3).t()), ValueError),
                      ({}, RuntimeError)]:          # everything in order but the device
        with pytest.raises(err):
            va.paged_kv_plan(**{**ok, **over})


def rope_ok(**over):
    return {**dict(q=torch.zeros(2, 4, 5, 64), k=torch.zeros(2, 2, 5, 64),
                   positions=torch.zeros(2, 5, dtype=torch.int64), inv_freq=torch.ones(32)), **over}


@pytest.mark.parametrize("over,err", [
    (dict(q=torch.zeros(4, 5, 64)), ValueError), (dict(k=torch.zeros(2, 2, 6, 64)), ValueError),
    (dict(k=torch.zeros(2, 2, 5, 32)), ValueError),
    (dict(k=torch.zeros(2, 2, 5, 64).half()), ValueError),
    (dict(q=torch.zeros(2, 4, 5, 64).double(), k=torch.zeros(2, 2, 5, 64).double()), TypeError),
    (dict(inv_freq=torch.ones(33)), ValueError), (dict(inv_freq=torch.ones(0)), ValueError),
    (dict(inv_freq=torch.ones(32).double()), ValueError),
    (dict(inv_freq=torch.ones(64)[::2]), ValueError),
    (dict(positions=torch.zeros(2, 4, dtype=torch.int64)), ValueError),
    (dict(positions=torch.zeros(2, 5)), TypeError),
    (dict(mrope_section=[16, 8]), ValueError), (dict(mrope_section=[40, -8]), ValueError),
    (dict(mrope_section=[16, 8, 8]), ValueError),  # positions of two rows, not of three axes
    (dict(mrope_section=[8, 8, 8, 4, 4], positions=torch.zeros(5, 2, 5, dtype=torch.int64)),
     ValueError),
    (dict(q_weight=torch.ones(32)), ValueError), (dict(q_weight=torch.ones(128)[::2]), ValueError),
    (dict(k_weight=torch.ones(64).half()), ValueError),
    (dict(q=torch.zeros(2, 0, 5, 64)), ValueError), (dict(k=torch.zeros(2, 0, 5, 64)), ValueError),
    ({}, RuntimeError)])
def test_rope_refusals(over, err):
    with pytest.raises(err):
        va.qk_norm_rope(**rope_ok(**over))


def store_ok(**over):
    return {**dict(q=torch.zeros(5, 4, 64), k=torch.zeros(5, 2, 64), v=torch.zeros(5, 2, 64),
                   k_cache=torch.zeros(3, 16, 2, 64), v_cache=torch.zeros(3, 16, 2, 64),
                   slot_mapping=torch.zeros(5, dtype=torch.int64),
                   positions=torch.zeros(5, dtype=torch.int64), inv_freq=torch.ones(32)), **over}


CACHE_ERRORS = [
    (dict(v=torch.zeros(5, 2, 32)), ValueError), (dict(v=torch.zeros(5, 2, 64).half()), ValueError),
    (dict(k=torch.zeros(2, 5, 2, 64)), ValueError),
    (dict(slot_mapping=torch.zeros(4, dtype=torch.int64)), ValueError),
    (dict(slot_mapping=i32(5)), ValueError),
    (dict(v_cache=torch.zeros(3, 16, 2, 32)), ValueError),
    (dict(k_cache=torch.zeros(3, 16, 4, 64), v_cache=torch.zeros(3, 16, 4, 64)), ValueError),
    (dict(kv_layout="HND"), ValueError), (dict(kv_layout="NDH"), KeyError),
    (dict(k_cache=torch.zeros(3, 16, 2, 64).half(), v_cache=torch.zeros(3, 16, 2, 64).half()),
     ValueError),
    (dict(k_cache=torch.zeros(0, 16, 2, 64), v_cache=torch.zeros(0, 16, 2, 64)), ValueError),
    (dict(k_cache=torch.zeros(3, 16, 64, 2).transpose(2, 3)), ValueError),
    ({}, RuntimeError)]


@pytest.mark.parametrize("over,err", CACHE_ERRORS + [
    (dict(q=torch.zeros(4, 4, 64)), ValueError), (dict(q=torch.zeros(5, 4, 64).half()), ValueError),
    (dict(q=torch.zeros(5, 0, 64)), ValueError),
    (dict(k=torch.zeros(5, 0, 64), v=torch.zeros(5, 0, 64), k_cache=torch.zeros(3, 16, 0, 64),
          v_cache=torch.zeros(3, 16, 0, 64)), ValueError),
    (dict(positions=torch.zeros(4, dtype=torch.int64)), ValueError)])
def test_rope_to_cache_refusals(over, err):
    with pytest.raises(err):
        va.qk_norm_rope_to_cache(**store_ok(**over))


@pytest.mark.parametrize("over,err", CACHE_ERRORS)
def test_write_refusals(over, err):
    args = store_ok(**over)
    for name in ("q", "positions", "inv_freq"):
        del args[name]
    with pytest.raises(err):
        va.write_paged_kv(**args)


@pytest.mark.parametrize("over,err", [
    (dict(q=torch.zeros(4, 64)), ValueError), (dict(q=torch.zeros(3, 5, 64)), ValueError),
    (dict(q=torch.zeros(3, 4, 32)), ValueError), (dict(q=torch.zeros(3, 4, 64).half()), ValueError),
    (dict(k_cache=torch.zeros(16, 2, 64)), ValueError),
    (dict(v_cache=torch.zeros(4, 16, 2, 64)), ValueError),
    (dict(block_tables=i32(2, 4)), ValueError), (dict(kv_lens=i32(3, 1)), ValueError),
    (dict(block_tables=torch.zeros(3, 4, dtype=torch.int64)), TypeError),
    (dict(kv_lens=torch.zeros(3, dtype=torch.int64)), TypeError),
    (dict(kv_layout="DNH"), KeyError), ({}, RuntimeError)])
def test_decode_refusals(over, err):
    args = {**dict(q=torch.zeros(3, 4, 64), k_cache=torch.zeros(3, 16, 2, 64),
                   v_cache=torch.zeros(3, 16, 2, 64), block_tables=i32(3, 4), kv_lens=i32(3)),
            **over}
    with pytest.raises(err):
        va.paged_decode_attention(**args)


@pytest.fixture(scope="module")
def L():
    if not os.path.exists(nat.LIB_PATH):
        from vecattention_amd import build
        build.build()
    return nat.lib()


P = 256  # an address that no refused call reads


def c_plan(L, **over):
    a = dict(kv=P, new=P, N=3, table=P, stn=4, M=4, free=P, F=5, head=None, page=16, tokens=8,
             out=P, indptr=P, slots=P, pos=P, req=P, taken=P, ws=None, wsb=0, stream=None)
    a.update(over)
    return L.va_paged_plan(*a.values())


def test_c_plan_errors(L):
    for over in (dict(kv=None), dict(table=None), dict(free=None), dict(slots=None),
                 dict(taken=None), dict(page=0), dict(page=2 ** 31), dict(N=-1), dict(M=-1),
                 dict(F=-1), dict(tokens=-1), dict(stn=3)):
        assert c_plan(L, **over) == nat.VA_ERR_ARG, over
    assert c_plan(L, N=2 ** 31) == nat.VA_ERR_UNSUPPORTED
    assert c_plan(L, tokens=2 ** 31) == nat.VA_ERR_UNSUPPORTED
    need = L.va_paged_plan_workspace_size(5000)
    assert need > 0 and L.va_paged_plan_workspace_size(5) == 0
    assert L.va_paged_plan_workspace_size(-1) == -1
    assert c_plan(L, N=5000) == nat.VA_ERR_WORKSPACE
    assert c_plan(L, N=5000, ws=P, wsb=need - 1) == nat.VA_ERR_WORKSPACE
    assert c_plan(L, N=5000, ws=P + 8, wsb=need) == nat.VA_ERR_ARG


def c_rope(L, **over):
    a = dict(dtype=1, q=P, a=0, b=64, c=64, k=P, d=0, e=64, f=64, qo=P, g=0, h=64, i=64, ko=P, j=0,
             l=64, m=64, B=1, Hq=4, Hk=2, S=8, D=64, pos=P, spa=0, spb=0, axes=1, sections=None,
             inv=P, rot=64, qw=None, kw=None, wt=1, eps=1e-6, scaling=1.0, inter=0, stream=None)
    a.update(over)
    return L.va_qk_norm_rope(*a.values())


def test_c_rope_errors(L):
    import ctypes
    for over in (dict(dtype=3), dict(q=None), dict(ko=None), dict(B=0), dict(S=0), dict(D=0),
                 dict(pos=None), dict(inv=None), dict(rot=0), dict(rot=33), dict(rot=66),
                 dict(axes=2), dict(axes=2, sections=(ctypes.c_int64 * 2)(16, 15)),
                 dict(axes=2, sections=(ctypes.c_int64 * 2)(33, -1)), dict(qw=P, wt=2)):
        assert c_rope(L, **over) == nat.VA_ERR_ARG, over
    for over in (dict(D=514), dict(axes=5), dict(S=2 ** 26), dict(B=2 ** 40, S=2 ** 40)):
        assert c_rope(L, **over) == nat.VA_ERR_UNSUPPORTED, over


def c_store(L, **over):
    a = dict(dtype=1, q=P, a=256, b=64, k=P, c=128, d=64, v=P, e=128, f=64, qo=P, g=256, h=64, kc=P,
             i=1, j=1, l=1, vc=P, m=1, n=1, o=1, pages=3, page=16, slots=P, T=5, Hq=4, Hk=2, D=64,
             pos=P, spa=0, axes=1, sections=None, inv=P, rot=64, qw=None, kw=None, wt=1, eps=1e-6,
             scaling=1.0, inter=0, stream=None)
    a.update(over)
    return L.va_qk_norm_rope_to_cache(*a.values())


def c_write(L, **over):
    a = dict(dtype=1, k=P, c=128, d=64, v=P, e=128, f=64, kc=P, i=1, j=1, l=1, vc=P, m=1, n=1, o=1,
             pages=3, page=16, slots=P, T=5, Hk=2, D=64, stream=None)
    a.update(over)
    return L.va_write_paged_kv(*a.values())


def test_c_store_and_write_errors(L):
    common = (dict(dtype=-1), dict(k=None), dict(v=None), dict(kc=None), dict(vc=None),
              dict(slots=None), dict(T=0), dict(Hk=0), dict(D=0), dict(pages=0), dict(page=0),
              dict(pages=2 ** 31), dict(page=2 ** 31))
    for call, more in ((c_write, ()), (c_store, (dict(q=None), dict(qo=None), dict(rot=66),
                                                 dict(pos=None)))):
        for over in common + more:
            assert call(L, **over) == nat.VA_ERR_ARG, (call, over)
    assert c_write(L, T=2 ** 24) == nat.VA_ERR_UNSUPPORTED
    assert c_write(L, Hk=2 ** 16, D=2 ** 16) == nat.VA_ERR_UNSUPPORTED
    assert c_store(L, T=2 ** 26) == nat.VA_ERR_UNSUPPORTED


def c_decode(L, **over):
    a = dict(dtype=1, q=P, a=512, b=128, k=P, c=4096, d=256, e=128, v=P, f=4096, g=256, h=128,
             out=P, i=512, j=128, table=P, stn=8, M=8, lens=P, N=3, Hq=4, Hk=2, D=128, page=16,
             pages=30, scale=0.1, ws=P, wsb=1 << 40, stream=None)
    a.update(over)
    return L.va_paged_decode_attn(*a.values())


def test_c_decode_errors(L):
    for over in (dict(dtype=9), dict(q=None), dict(out=None), dict(table=None), dict(lens=None),
                 dict(N=0), dict(Hq=0), dict(D=0), dict(M=-1), dict(Hq=5), dict(page=0),
                 dict(pages=0), dict(ws=P + 8)):
        assert c_decode(L, **over) == nat.VA_ERR_ARG, over
    for over in (dict(D=257), dict(N=2 ** 22), dict(N=1000, M=2 ** 27), dict(M=2 ** 31),
                 dict(M=2 ** 31 - 1, page=2 ** 31 - 1)):
        assert c_decode(L, **over) == nat.VA_ERR_UNSUPPORTED, over
    need = L.va_paged_decode_workspace_size(1, 3, 4, 2, 128, 8, 16)
    assert need > 0
    assert c_decode(L, ws=None) == nat.VA_ERR_WORKSPACE
    assert c_decode(L, wsb=need - 1) == nat.VA_ERR_WORKSPACE
    assert L.va_paged_decode_workspace_size(1, 3, 5, 2, 128, 8, 16) == -1


def test_operators_have_no_backward():
    """Refused after the device, so on the CPU the device speaks first; on a GPU
    test_gpu_paged.py sees it."""
    w = torch.ones(64, requires_grad=True)
    with pytest.raises(RuntimeError, match="GPU"):
        va.qk_norm_rope(**rope_ok(q_weight=w))


def test_arguments_that_are_no_tensors_or_numbers():
    with pytest.raises(TypeError, match="k must be a tensor"):
        va.qk_norm_rope(**rope_ok(k=[1.0]))
    with pytest.raises(TypeError, match="q_weight must be a tensor"):
        va.qk_norm_rope(**rope_ok(q_weight=3))
    with pytest.raises(TypeError):
        va.qk_norm_rope(**rope_ok(mrope_section=7))
    with pytest.raises(TypeError):
        va.qk_norm_rope(**rope_ok(mrope_section=[16.5, 8, 8]))
    with pytest.raises(TypeError):
        va.paged_kv_plan(i32(3), i32(3), i32(3, 4), i32(5), 16.5, 8)
    with pytest.raises(OverflowError):
        va.paged_kv_plan(i32(3), i32(3), i32(3, 4), i32(5), 16, 1 << 70)
    with pytest.raises(TypeError, match="arguments"):
        nat._host_module().plan(1, 2)
    with pytest.raises(KeyError):
        va.write_paged_kv(torch.zeros(5, 2, 64), torch.zeros(5, 2, 64), torch.zeros(3, 16, 2, 64),
                          torch.zeros(3, 16, 2, 64), torch.zeros(5, dtype=torch.int64), None)


def test_operators_have_no_forward_derivative():
    """A tangent is refused, not dropped; where forward mode is off, the device speaks next."""
    from torch.autograd import forward_ad as fw
    x, kc, slots = torch.ones(5, 2, 64), torch.zeros(3, 16, 2, 64), torch.zeros(5, dtype=torch.int64)
    inv, w = torch.ones(32), torch.ones(64)
    table, lens = torch.zeros(5, 1, dtype=torch.int32), torch.ones(5, dtype=torch.int32)
    calls = [(lambda q, k, f, u, v: va.qk_norm_rope(q[None], k[None], slots[:2], f, u, v),
              [x, x, inv, w, w]),
             (lambda q, k, v, c, d, f, u: va.qk_norm_rope_to_cache(q, k, v, c, d, slots, slots, f,
                                                                   u, u),
              [x, x, x, kc, kc, inv, w]),
             (lambda k, v, c, d: va.write_paged_kv(k, v, c, d, slots), [x, x, kc, kc]),
             (lambda k: va.write_paged_kv(k[..., ::2], x[..., ::2], kc[..., :32], kc[..., :32],
                                          slots), [x]),  # a copied one
             (lambda q, c, d: va.paged_decode_attention(q, c, d, table, lens), [x, kc, kc])]
    with fw.dual_level():
        for call, args in calls:
            for i, a in enumerate(args):
                dual = [fw.make_dual(b, torch.ones_like(b)) if i == j else b
                        for j, b in enumerate(args)]
                with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                    call(*dual)
                with fw._set_fwd_grad_enabled(False), pytest.raises(RuntimeError, match="the GPU"):
                    call(*dual)
            with pytest.raises(RuntimeError, match="the GPU"):
                call(*args)


@pytest.mark.parametrize("bad", [None, [1.0], 3, "q"])
def test_a_first_argument_that_is_no_tensor(bad):
    """It chooses the GPU that the call runs on, and is refused as the others are."""
    x, kc, slots, inv = (torch.zeros(5, 2, 64), torch.zeros(3, 16, 2, 64),
                         torch.zeros(5, dtype=torch.int64), torch.ones(32))
    for name, call in [
            ("block_tables", lambda: va.paged_kv_plan(i32(3), i32(3), bad, i32(5), 16, 8)),
            ("q", lambda: va.qk_norm_rope(bad, x[None], slots, inv)),
            ("q", lambda: va.qk_norm_rope_to_cache(bad, x, x, kc, kc, slots, slots, inv)),
            ("k", lambda: va.write_paged_kv(bad, x, kc, kc, slots)),
            ("q", lambda: va.paged_decode_attention(bad, kc, kc, i32(5, 1), i32(5)))]:
        with pytest.raises(TypeError, match=f"^{name} must be a tensor"):
            call()


def test_the_documented_step_rotates_by_the_models_positions(monkeypatch):
    """The documentation's step of a prompt with an image and of generated tokens, run with
    recorders in place of the operators: a generated token's position is the one behind the
    prompt's last, not its index."""
    import glob
    import re
    blocks = [b for f in sorted(glob.glob(os.path.join(os.path.dirname(HERE), "*.md")))
              for b in re.findall(r"```python\n(.*?)```", open(f).read(), re.S)
              if "= paged_decode_attention(" in b]
    assert len(blocks) == 1
    N, S, i = 3, 36, 1
    rotated = []

    def plan(kv_lens, new_lens, tables, free_pages, page, num_tokens, head=None):
        index = torch.full((N,), S)        # each request's next token, and one row of padding
        return va.PagedStep(kv_lens, None, torch.cat([index, index[:1] * 0 - 1]),
                            torch.cat([index, index[:1] * 0]),
                            torch.tensor([0, 1, 2, -1], dtype=torch.int32), None)

    def rotate(q, k, v, kc, vc, slots, positions, *more, **options):
        rotated.append((positions, more, options))
        return q

    monkeypatch.setattr(va, "paged_kv_plan", plan)
    monkeypatch.setattr(va, "qk_norm_rope", lambda q, k, *more, **options: (q, k))
    monkeypatch.setattr(va, "qk_norm_rope_to_cache", rotate)
    for name in ("write_paged_kv", "paged_decode_attention", "VecAttention_prefill"):
        monkeypatch.setattr(va, name, lambda *args, **options: None)
    # Five tokens of text, an image of 4 x 6, seven tokens of text behind its largest position.
    at = torch.cat([torch.arange(5).expand(3, 5),
                    5 + torch.stack([torch.zeros(24).long(), torch.arange(24) // 6,
                                     torch.arange(24) % 6]),
                    11 + torch.arange(7).expand(3, 7)], 1)[:, None]
    x = torch.zeros(1, 2, S, 64)
    exec(blocks[0].replace('"cuda"', '"cpu"'), dict(
        torch=torch, num_pages=8, Hk=2, D=64, N=N, max_pages=4, i=i, num_tokens=N + 1, q=x, k=x,
        v=x, kv_lens=None, new_lens=None, position_ids=at, q_norm=None, k_norm=None,
        inv_freq=torch.ones(32), rotary_emb=type("", (), {"inv_freq": torch.ones(32)})))
    (positions, _, options), = rotated
    want = [S] * N
    want[i] = int(at.max()) + 1
    assert positions[:N].tolist() == want and "mrope_section" not in options
