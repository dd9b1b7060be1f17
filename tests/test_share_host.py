"""The operators on pages that rows share, without a GPU: the plain forms by hand, the
index arithmetic (a host build of csrc/paged.h), and every refusal."""
import os
import random
import shutil
import subprocess

import pytest
import torch

import share_reference as ref
import vecattention_amd as va
from vecattention_amd import _native as nat

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "vecattention_amd", "csrc")


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def test_plain_fork_by_hand():
    # Two beams behind a shared page 3; the second one is dropped, the first forked.
    lens, table, shares, free, head, src, dst, rows = ref.fork(
        [6, 7], [0, 0], [[3, 5, -1], [3, 6, -1]], [0, 0, 0, 1, 0, 0, 0, 0], [9, 9, 4, 7], 4, 2)
    assert lens == [6, 6] and table == [[3, 5, -1], [3, 6, -1]]     # 6 was freed and taken again
    assert shares == [0, 0, 0, 1, 0, 0, 0, 0] and free == [9, 9, 4, 7] and head == 2
    assert src == [-1, 5] and dst == [-1, 6] and rows == [0, 2]
    # Cut back into the shared page: both write to it, so the second gets one of its own.
    lens, table, shares, free, head, src, dst, rows = ref.fork(
        [6, 7], [0, 1], [[3, 5, -1], [3, 6, -1]], [0, 0, 0, 1, 0, 0, 0, 0], [9, 9, 4, 7], 4, 2,
        [2, 3])
    assert lens == [2, 3] and table == [[3, -1, -1], [5, -1, -1]] and free == [9, 6, 4, 7]
    assert shares == [0] * 8 and head == 1 and (src, dst, rows) == ([-1, 3], [-1, 5], [0, 3])
    # All dropped: the pages return in ascending order.
    out = ref.fork([6, 7], [], [[3, 5, -1], [3, 6, -1]], [0, 0, 0, 1, 0, 0, 0, 0], [9, 9, 9], 4, 3)
    assert out[3] == [3, 5, 6] and out[4] == 0
    # A row that has the page whole keeps it; the one that writes to it gets another.
    out = ref.fork([4, 4], [0, 1], [[3], [3]], [0, 0, 0, 1], [0, 1], 4, 0, [4, 2])
    assert out[1] == [[3], [0]] and out[2] == [0] * 4 and out[4] == 1


def test_plain_compaction_and_prefix_by_hand():
    table, shares, free, head, src, dst, moves = ref.compact(
        [5, 3], [[6, 2, -1], [7, 9, 9]], [0, 0, 1, 0, 0, 0, 2, 3, 0, 0], [8, 4, 0, 3, 99], 4, 1)
    # In the tables 2, 6, 7; free 0, 3, 4: the lowest three are 0, 2, 3.
    assert table == [[0, 2, -1], [3, 9, 9]]
    assert (src, dst) == ([6, 7, -1, -1, -1], [0, 3, -1, -1, -1])
    assert shares == [2, 0, 1, 3, 0, 0, 0, 0, 0, 0] and moves == 2
    assert head == 2 and free == [8, 4, 4, 6, 7]
    lens, table = [9, 8, 0, 12, 12, 3], [[1, 2, 5], [1, 2, 6], [1, 2, 5], [1, 2, 7], [1, 3, 7],
                                         [1, 2, 7]]
    assert ref.prefix(lens, table, 4) == ([8, 8, 0, 0, 0, 0], [2, 0, 0, 0, 0, 0])
    assert ref.prefix(lens, table, 4, [5, 5, 5, 5, 5, 6]) == ([8, 8, 0, 4, 4, 0],
                                                              [2, 0, 0, 2, 0, 0])


def test_plain_fork_keeps_pages_apart():
    """Over random steps: a page that a row will write to is its own, every page is held or
    free, and the shares are the holders less one."""
    r = random.Random(3)
    page, width, P = 4, 9, 120
    lens, table, shares = [0] * 3, [[-1] * width for _ in range(3)], [0] * P
    free, head = list(range(P)), 0
    for step in range(60):
        for n in range(len(lens)):  # what the plan does: some tokens more
            add = r.randint(0, 5)
            end = min(lens[n] + add, width * page)
            for k in range(ref.pages_of(lens[n], page, width), ref.pages_of(end, page, width)):
                table[n][k] = free[head]
                head += 1
            lens[n] = end
        parents = [r.randint(-1, len(lens) - 1) for _ in range(r.randint(1, 6))]
        keep = [r.randint(0, 40) for _ in parents] if r.random() < 0.5 else None
        lens, table, shares, free, head, src, dst, rows = ref.fork(
            lens, parents, table, shares, free, page, head, keep)
        holders = {}
        for n, row in enumerate(table):
            for k in range(ref.pages_of(lens[n], page, width)):
                holders.setdefault(row[k], []).append((n, k))
        assert sorted(list(holders) + free[head:]) == list(range(P))
        for p in range(P):
            assert shares[p] == max(len(holders.get(p, [])) - 1, 0)
        for n, row in enumerate(table):
            if lens[n] % page:
                assert holders[row[lens[n] // page]] == [(n, lens[n] // page)]
        for a, b, c in zip(src, dst, rows):
            assert (a in holders and len(holders[b]) == 1 and 0 < c < page) if b >= 0 else c == 0


PROG = r"""
#include "paged.h"
#include <cstdio>
int main() {
  using namespace va;
  if (held_pages(-1, 16, 4) || held_pages(0, 16, 4) || held_pages(1, 16, 4) != 1 ||
      held_pages(16, 16, 4) != 1 || held_pages(17, 16, 4) != 2 || held_pages(999, 16, 4) != 4 ||
      held_pages(0x7fffffff, 1, 0x7fffffff) != 0x7fffffff || held_pages(5, 0x7fffffff, 3) != 1 ||
      held_pages(9, 4, 0)) { printf("BAD held\n"); return 1; }
  if (open_page(0, 16, 4) != -1 || open_page(16, 16, 4) != -1 || open_page(17, 16, 4) != 1 ||
      open_page(63, 16, 4) != 3 || open_page(65, 16, 4) != -1 || open_page(-3, 16, 4) != -1 ||
      open_page(7, 1, 100) != -1 || open_page(0x7fffffff, 2, 0x7fffffff) != 0x3fffffff ||
      open_page(3, 4, 0) != -1) { printf("BAD open\n"); return 1; }
  if (is_page(-1, 5) || is_page(5, 5) || !is_page(0, 5) || !is_page(4, 5) || is_page(0, 0)) {
    printf("BAD page\n"); return 1; }
  printf("OK\n");
  return 0;
}
"""


def test_index_arithmetic(tmp_path):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("no hipcc")
    src, exe = tmp_path / "share.cpp", tmp_path / "share"
    src.write_text(PROG)
    subprocess.run([hipcc, "-x", "hip", "--offload-arch=gfx950", "-O2", "-std=c++17", "-I", CSRC,
                    "-o", str(exe), str(src)], check=True, capture_output=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0 and out.stdout.strip() == "OK", out.stdout + out.stderr


def fork_ok(**over):
    return {**dict(kv_lens=i32(3), parents=i32(5), block_tables=i32(3, 4), page_shares=i32(9),
                   free_pages=i32(9), page_size=16), **over}


POOL_ERRORS = [
    (dict(kv_lens=i32(3, 1)), ValueError), (dict(block_tables=i32(2, 4)), ValueError),
    (dict(block_tables=i32(3)), ValueError), (dict(page_shares=i32(9, 1)), ValueError),
    (dict(free_pages=i32(9, 1)), ValueError), (dict(free_head=i32(2)), ValueError),
    (dict(kv_lens=torch.zeros(3)), TypeError),
    (dict(page_shares=torch.zeros(9, dtype=torch.int64)), TypeError),
    (dict(block_tables=torch.zeros(3, 4, dtype=torch.int64)), TypeError),
    (dict(free_head=torch.zeros(1, dtype=torch.int64)), TypeError),
    (dict(page_size=0), ValueError), (dict(page_size=-16), ValueError),
    (dict(page_size=16.5), TypeError), (dict(page_shares=[0, 0]), TypeError),
    (dict(free_head=3), TypeError), ({}, RuntimeError)]


@pytest.mark.parametrize("over,err", POOL_ERRORS + [
    (dict(parents=i32(5, 1)), ValueError), (dict(parents=torch.zeros(5)), TypeError),
    (dict(keep_lens=i32(4)), ValueError), (dict(parents=None), TypeError),
    (dict(keep_lens=torch.zeros(5, dtype=torch.int64)), TypeError)])
def test_fork_refusals(over, err):
    with pytest.raises(err):
        va.paged_kv_fork(**fork_ok(**over))


@pytest.mark.parametrize("over,err", POOL_ERRORS)
def test_compact_refusals(over, err):
    args = fork_ok(**over)
    del args["parents"]
    with pytest.raises(err):
        va.paged_kv_compact(**args)


@pytest.mark.parametrize("over,err", [
    (dict(kv_lens=i32(3, 1)), ValueError), (dict(block_tables=i32(2, 4)), ValueError),
    (dict(group_ids=i32(2)), ValueError), (dict(page_size=0), ValueError),
    (dict(group_ids=torch.zeros(3)), TypeError), (dict(kv_lens=torch.zeros(3)), TypeError),
    (dict(kv_lens=[1, 2, 3]), TypeError), ({}, RuntimeError)])
def test_prefix_refusals(over, err):
    with pytest.raises(err):
        va.paged_kv_prefix(**{**dict(kv_lens=i32(3), block_tables=i32(3, 4), page_size=16), **over})


def cache(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("over,err", [
    (dict(src_pages=i32(3)), ValueError), (dict(src_pages=i32(4, 1)), ValueError),
    (dict(rows=i32(5)), ValueError), (dict(rows=torch.zeros(4)), TypeError),
    (dict(dst_pages=torch.zeros(4, dtype=torch.int64)), TypeError),
    (dict(k_caches=[]), ValueError), (dict(v_caches=[]), ValueError),
    (dict(k_caches=[cache(3, 16, 2, 64)] * 2), ValueError),
    (dict(k_caches=[cache(3, 16, 2, 64)] * 2, v_caches=[cache(3, 16, 2, 64),
                                                       cache(4, 16, 2, 64)]), ValueError),
    (dict(k_caches=[cache(3, 16, 2, 64), cache(3, 2, 16, 64).transpose(1, 2)],
          v_caches=[cache(3, 16, 2, 64)] * 2), ValueError),
    (dict(k_caches=[cache(3, 16, 2, 64), cache(3, 16, 2, 64, dtype=torch.float16)],
          v_caches=[cache(3, 16, 2, 64)] * 2), ValueError),
    (dict(v_caches=cache(3, 16, 2, 32)), ValueError), (dict(k_caches=cache(16, 2, 64)), ValueError),
    (dict(k_caches=cache(3, 16, 2, 64).double(), v_caches=cache(3, 16, 2, 64).double()), TypeError),
    (dict(v_caches=cache(3, 16, 2, 64).half()), ValueError),
    (dict(k_caches=cache(0, 16, 2, 64), v_caches=cache(0, 16, 2, 64)), ValueError),
    (dict(k_caches=cache(3, 16, 64, 2).transpose(2, 3)), ValueError),
    (dict(kv_layout="NDH"), KeyError), (dict(k_caches=3), TypeError),
    (dict(v_caches="v"), TypeError),
    (dict(k_caches=[3], v_caches=[4]), TypeError), ({}, RuntimeError)])
def test_copy_refusals(over, err):
    with pytest.raises(err):
        va.copy_paged_kv(**{**dict(k_caches=cache(3, 16, 2, 64), v_caches=cache(3, 16, 2, 64),
                                   src_pages=i32(4), dst_pages=i32(4)), **over})


def attend_ok(**over):
    return {**dict(q=torch.zeros(3, 4, 64), k_cache=torch.zeros(3, 16, 2, 64),
                   v_cache=torch.zeros(3, 16, 2, 64), block_tables=i32(3, 4), kv_lens=i32(3),
                   prefix=(i32(3), i32(3))), **over}


@pytest.mark.parametrize("over,err", [
    (dict(q=torch.zeros(4, 64)), ValueError), (dict(q=torch.zeros(3, 5, 64)), ValueError),
    (dict(q=torch.zeros(3, 4, 32)), ValueError), (dict(q=torch.zeros(3, 4, 64).half()), ValueError),
    (dict(k_cache=torch.zeros(16, 2, 64)), ValueError),
    (dict(block_tables=i32(2, 4)), ValueError), (dict(kv_lens=i32(3, 1)), ValueError),
    (dict(block_tables=torch.zeros(3, 4, dtype=torch.int64)), TypeError),
    (dict(prefix=(i32(2), i32(3))), ValueError), (dict(prefix=(i32(3), i32(3, 1))), ValueError),
    (dict(prefix=(i32(3), torch.zeros(3))), TypeError), (dict(prefix=(i32(3), None)), TypeError),
    (dict(prefix=(i32(3),)), ValueError), (dict(prefix=None), TypeError),
    (dict(kv_layout="DNH"), KeyError), ({}, RuntimeError)])
def test_attend_refusals(over, err):
    with pytest.raises(err):
        va.paged_prefix_decode_attention(**attend_ok(**over))


def test_no_forward_derivative():
    from torch.autograd import forward_ad as fw
    x, kc = torch.ones(3, 4, 64), torch.zeros(3, 16, 2, 64)
    calls = [(lambda q, c, d: va.paged_prefix_decode_attention(**attend_ok(q=q, k_cache=c,
                                                                           v_cache=d)),
              [x, kc, kc]),
             (lambda c, d: va.copy_paged_kv([kc, c], [kc, d], i32(4), i32(4)), [kc, kc])]
    with fw.dual_level():
        for call, args in calls:
            for i, a in enumerate(args):
                dual = [fw.make_dual(b, torch.ones_like(b)) if i == j else b
                        for j, b in enumerate(args)]
                with torch.no_grad(), pytest.raises((NotImplementedError, RuntimeError)):
                    call(*dual)


@pytest.fixture(scope="module")
def L():
    if not os.path.exists(nat.LIB_PATH):
        from vecattention_amd import build
        build.build()
    return nat.lib()


P = 256  # an address that no refused call reads


def c_fork(L, **over):
    a = dict(kv=P, keep=None, parents=P, N=3, R=5, table=P, stn=4, M=4, shares=P, pages=9, free=P,
             F=9, head=None, page=16, kvo=P, to=P, so=P, fo=P, ho=P, src=P, dst=P, rows=P, ws=P,
             wsb=1 << 30, stream=None)
    a.update(over)
    return L.va_paged_fork(*a.values())


def test_c_fork_errors(L):
    for over in (dict(kv=None), dict(parents=None), dict(table=None), dict(shares=None),
                 dict(free=None), dict(kvo=None), dict(to=None), dict(so=None), dict(fo=None),
                 dict(ho=None), dict(src=None), dict(dst=None), dict(rows=None), dict(N=-1),
                 dict(R=-1), dict(M=-1), dict(pages=-1), dict(F=-1), dict(page=0),
                 dict(page=2 ** 31), dict(stn=-1), dict(ws=P + 8)):
        assert c_fork(L, **over) == nat.VA_ERR_ARG, over
    for over in (dict(N=65537), dict(R=65537), dict(M=2 ** 31), dict(pages=2 ** 31),
                 dict(F=2 ** 31), dict(R=65536, N=65536, M=2 ** 24)):
        assert c_fork(L, **over) == nat.VA_ERR_UNSUPPORTED, over
    need = L.va_paged_fork_workspace_size(5, 9)
    assert need > 0 and L.va_paged_fork_workspace_size(-1, 9) == -1
    assert L.va_paged_fork_workspace_size(5, -1) == -1
    assert c_fork(L, ws=None) == nat.VA_ERR_WORKSPACE
    assert c_fork(L, wsb=need - 1) == nat.VA_ERR_WORKSPACE


def c_compact(L, **over):
    a = dict(kv=P, N=3, table=P, stn=4, M=4, shares=P, pages=9, free=P, F=9, head=None, page=16,
             to=P, so=P, fo=P, ho=P, src=P, dst=P, moves=P, ws=P, wsb=1 << 30, stream=None)
    a.update(over)
    return L.va_paged_compact(*a.values())


def test_c_compact_errors(L):
    for over in (dict(kv=None), dict(table=None), dict(shares=None), dict(free=None), dict(to=None),
                 dict(so=None), dict(fo=None), dict(ho=None), dict(src=None), dict(dst=None),
                 dict(moves=None), dict(N=-1), dict(M=-1), dict(pages=-1), dict(page=0),
                 dict(ws=P + 8)):
        assert c_compact(L, **over) == nat.VA_ERR_ARG, over
    for over in (dict(N=2 ** 30), dict(N=2 ** 22, M=4096), dict(M=2 ** 31), dict(pages=2 ** 31)):
        assert c_compact(L, **over) == nat.VA_ERR_UNSUPPORTED, over
    need = L.va_paged_compact_workspace_size(9)
    assert need > 0 and L.va_paged_compact_workspace_size(-1) == -1
    assert c_compact(L, wsb=need - 1) == nat.VA_ERR_WORKSPACE


def c_prefix(L, **over):
    a = dict(kv=P, N=3, table=P, stn=4, M=4, ids=None, page=16, lens=P, rows=P, ws=P, wsb=1 << 20,
             stream=None)
    a.update(over)
    return L.va_paged_prefix(*a.values())


def test_c_prefix_errors(L):
    for over in (dict(kv=None), dict(table=None), dict(lens=None), dict(rows=None), dict(N=-1),
                 dict(M=-1), dict(page=0), dict(ws=P + 8)):
        assert c_prefix(L, **over) == nat.VA_ERR_ARG, over
    assert c_prefix(L, N=65537) == nat.VA_ERR_UNSUPPORTED
    need = L.va_paged_prefix_workspace_size(3)
    assert need > 0 and L.va_paged_prefix_workspace_size(-1) == -1
    assert c_prefix(L, wsb=need - 1) == nat.VA_ERR_WORKSPACE
    assert c_prefix(L, N=0, kv=None) == nat.VA_OK


def c_copy(L, **over):
    import ctypes
    two = (ctypes.c_void_p * 2)(P, P)
    a = dict(dtype=1, k=two, v=two, layers=2, a=1, b=1, c=1, d=1, e=1, f=1, pages=9, page=16, Hk=2,
             D=64, src=P, dst=P, rows=None, C=3, stream=None)
    a.update(over)
    return L.va_copy_paged_kv(*a.values())


def test_c_copy_errors(L):
    import ctypes
    hole = (ctypes.c_void_p * 2)(P, None)
    for over in (dict(dtype=7), dict(k=None), dict(v=None), dict(k=hole), dict(v=hole),
                 dict(layers=-1), dict(C=-1), dict(Hk=0), dict(D=0), dict(a=-1), dict(f=-1),
                 dict(pages=0), dict(pages=2 ** 31), dict(page=0), dict(src=None), dict(dst=None)):
        assert c_copy(L, **over) == nat.VA_ERR_ARG, over
    for over in (dict(C=2 ** 31), dict(Hk=2 ** 16, D=2 ** 16), dict(page=2 ** 30, Hk=8),
                 dict(page=2 ** 20, Hk=16, C=2 ** 30)):
        assert c_copy(L, **over) == nat.VA_ERR_UNSUPPORTED, over
    assert c_copy(L, C=0) == nat.VA_OK and c_copy(L, layers=0) == nat.VA_OK


def c_attend(L, **over):
    a = dict(dtype=1, q=P, a=512, b=128, k=P, c=4096, d=256, e=128, v=P, f=4096, g=256, h=128,
             out=P, i=512, j=128, table=P, stn=8, M=8, lens=P, prefix=P, group=P, N=3, Hq=4, Hk=2,
             D=128, page=16, pages=30, scale=0.1, ws=P, wsb=1 << 40, stream=None)
    a.update(over)
    return L.va_paged_prefix_decode_attn(*a.values())


def test_c_attend_errors(L):
    for over in (dict(dtype=9), dict(q=None), dict(out=None), dict(table=None), dict(lens=None),
                 dict(prefix=None), dict(group=None), dict(N=0), dict(Hq=0), dict(D=0), dict(M=-1),
                 dict(Hq=5), dict(page=0), dict(pages=0), dict(ws=P + 8)):
        assert c_attend(L, **over) == nat.VA_ERR_ARG, over
    for over in (dict(D=257), dict(N=2 ** 22), dict(N=1000, M=2 ** 27), dict(M=2 ** 31)):
        assert c_attend(L, **over) == nat.VA_ERR_UNSUPPORTED, over
    need = L.va_paged_prefix_decode_workspace_size(1, 3, 4, 2, 128, 8, 16)
    assert need > 0
    assert c_attend(L, ws=None) == nat.VA_ERR_WORKSPACE
    assert c_attend(L, wsb=need - 1) == nat.VA_ERR_WORKSPACE
    assert L.va_paged_prefix_decode_workspace_size(1, 3, 5, 2, 128, 8, 16) == -1


def test_no_matrix_result_of_shared_prefixes_is_read_too_soon(tmp_path, monkeypatch):
    import asm_hazards
    # Passes + 3 for 16-bit operands, of which 32x32x16 takes 8; passes + 2 for fp32 ones, of which
    # 32x32x2 takes 16.
    monkeypatch.setattr(asm_hazards, "NEED", {**asm_hazards.NEED, "v_mfma_f32_32x32x16_bf16": 11,
                                              "v_mfma_f32_32x32x16_f16": 11,
                                              "v_mfma_f32_32x32x2_f32": 18})
    from vecattention_amd import build
    csrc = os.path.join(os.path.dirname(build.__file__), "csrc")
    out = tmp_path / "paged_prefix.s"
    subprocess.run([build.hipcc(), *build.FLAGS, "--cuda-device-only", "-S",
                    os.path.join(csrc, "paged_prefix.hip"), "-o", str(out)], check=True,
                   capture_output=True)
    count, early = asm_hazards.early_reads(out.read_text())
    assert count > 300 and early == []
