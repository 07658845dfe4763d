"""The paged key-value cache: append with norm and rotation, attention of new tokens, eviction.

CPU: the address and bounds arithmetic the kernels use (csrc/kv_pages.h, compiled for the host), the
oracle's eviction on a hand-made case, and what the C entries refuse. GPU: every call against
oracle/streaming.py in float64 on copies of the same cache, in pools whose unused slots hold NaN.

Bounds for attention, from u = finfo.eps / 2 of the 16-bit type: P is rounded to that type for its
product (u of sum p|v|; in fp16 also half a subnormal step, 2^-25, of sum |v|), O once more (u of |o|).
A score is a float32 sum of D products and a scaling, off by at most es = (D + 8) 2^-24 of the largest
scaled sum |q k| of its row, which moves each p by the factor 1 +- 2 es; exponentials, sums and joins add less than
64 half steps of float32.
"""
import ctypes
import math
import os
import subprocess

import pytest
import torch

from oracle import streaming as st

F32 = 2.0 ** -24
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


# ---------------------------------------------------------------- on the CPU


def test_addresses_stay_inside_the_pool(tmp_path):
    """Whatever table, lengths and slots hold: a located slot lies on a page of the pool, lengths are
    clipped to the capacity, and appended slots stay below it."""
    src = tmp_path / "pages.cpp"
    src.write_text(r"""
#include <climits>
#include <cstdio>
#include <vector>
#include "kv_pages.h"
using namespace dmad;
int main() {
  const int ids[] = {-1, 0, 1, 5, 6, 7, INT_MAX, INT_MIN, -7};
  const int nums[] = {0, 1, 15, 16, 17, 47, 48, 95, 96, 97, 143, 144, 145, INT_MAX, INT_MAX - 1, INT_MIN, -1, -16};
  long checked = 0;
  for (int P : {16, 48}) for (int M : {0, 1, 3}) {
    const int N = 6, H = 2, B = 2;
    std::vector<int32_t> table(B * (M + 1)), lengths(B), seen(B);
    KvPages kv{};
    kv.table = table.data(); kv.table_stride = M + 1; kv.lengths = lengths.data(); kv.seen = seen.data();
    kv.num_pages = N; kv.heads = H; kv.B = B; kv.set_pages(P, M);
    kv.k_sp = kv.v_sp = H * P * 16; kv.k_sh = kv.v_sh = P * 16; kv.k_sl = kv.v_sl = 16;
    for (int id : ids) {
      for (auto& t : table) t = id;
      for (int n : nums) {
        lengths[0] = lengths[1] = n;
        const int len = kv.length(1);
        if (len < 0 || len > M * P || (n >= 0 && n <= M * P && len != n)) return 1;
        for (int s : nums) {
          const KvSlot at = kv.locate(1, s);
          const bool should = s >= 0 && s < M * P && id >= 0 && id < N;
          if (should != (at.page >= 0)) return 2;
          if (should && (at.page != id || at.slot != s % P)) return 3;
          if (should && (kv.index(at, H - 1) < 0 || kv.index(at, H - 1) >= (int64_t)N * H * P)) return 4;
          if (should && (kv.k_offset(at, H - 1) + 16 > (int64_t)N * H * P * 16 || kv.v_offset(at, 0) < 0)) return 5;
          if (!should && (at.page != -1 || at.slot != 0)) return 6;
          if (s >= 0) {
            const int slot = kv_append_slot(len, s, M * P);
            if (slot != -1 && (slot < len || slot >= M * P || slot - len != s)) return 7;
            if (slot == -1 && (int64_t)len + s < (int64_t)M * P) return 8;
            const int after = kv_append_length(len, s, M * P);
            if (after < len || after > M * P || (after < M * P && after - len != s)) return 9;
          }
          ++checked;
        }
      }
    }
  }
  // offsets beyond 32 bits
  KvPages big{};
  int32_t page = 70000;
  big.table = &page; big.table_stride = 1; big.num_pages = 100000; big.heads = 8; big.B = 1; big.set_pages(64, 1);
  big.k_sp = big.v_sp = 8 * 64 * 128; big.k_sh = big.v_sh = 64 * 128; big.k_sl = big.v_sl = 128;
  if (big.k_offset(big.locate(0, 63), 7) != 70000LL * 65536 + 7 * 8192 + 63 * 128) return 10;
  // the quotient by the page size, at its steps and at the largest slot
  for (int P = 16; P <= 1 << 26; P += P < 4096 ? 16 : P % 32 ? 16 : P / 3 / 16 * 16) {
    const int M = (1 << 26) / P;
    std::vector<int32_t> pages(M);
    for (int i = 0; i < M; ++i) pages[i] = i;
    KvPages kv{};
    kv.table = pages.data(); kv.num_pages = M; kv.B = 1; kv.set_pages(P, M);
    for (int i = 0; i < M; i = i < 100 ? i + 1 : i + 1 + i / 7) {
      const KvSlot a = kv.locate(0, i * P), z = kv.locate(0, i * P + P - 1);
      if (a.page != i || a.slot != 0 || z.page != i || z.slot != P - 1) return 11;
      ++checked;
    }
    if (kv.locate(0, M * P - 1).page != M - 1) return 12;
  }
  printf("%ld\n", checked);
  return 0;
}
""")
    exe = tmp_path / "pages"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover",
                    "-I", os.path.join(ROOT, "dmad_amd", "csrc"), str(src), "-o", str(exe)], check=True)
    done = subprocess.run([str(exe)], capture_output=True, text=True)
    assert done.returncode == 0 and int(done.stdout) > 1000, (done.returncode, done.stderr)


def test_oracle_eviction_by_hand():
    """Six slots, four stay: the sink 0, the two last positions (4 and 5) and the heavier of 1, 2, 3."""
    c = dict(k_pages=torch.arange(16.0).view(1, 1, 16, 1).expand(1, 1, 16, 16).clone(), v_pages=torch.zeros(1, 1, 16, 16),
             page_table=torch.zeros(1, 1, dtype=torch.int32), lengths=torch.tensor([6]), seen=torch.tensor([6]),
             weight=torch.tensor([0.0, 1.0, 3.0, 1.0, 0.0, 0.0] + [9.0] * 10).view(1, 1, 16),
             position=torch.arange(16).view(1, 1, 16))
    st.evict(c, 4, recent=2, sink=1)
    assert c["lengths"].tolist() == [4]
    assert c["position"][0, 0, :6].tolist() == [0, 4, 2, 5, 4, 5]
    assert c["k_pages"][0, 0, :4, 0].tolist() == [0, 4, 2, 5] and c["weight"][0, 0, :4].tolist() == [0, 0, 3, 0]


def test_oracle_attention_matches_loops():
    g = torch.Generator().manual_seed(0)
    c = dict(k_pages=torch.randn(3, 1, 16, 16, generator=g), v_pages=torch.randn(3, 1, 16, 16, generator=g),
             page_table=torch.tensor([[2, 0]], dtype=torch.int32), lengths=torch.tensor([20]), seen=torch.tensor([20]),
             weight=torch.zeros(3, 1, 16), position=torch.zeros(3, 1, 16, dtype=torch.int32))
    q = torch.randn(1, 2, 2, 16, generator=g)
    o, lse, _ = st.attend(c, q, causal=True, accumulate=True)
    for i in range(2):
        for h in range(2):
            rows = [(2, s) for s in range(16)] + [(0, s) for s in range(3 + i)]
            s = [sum(float(q[0, i, h, d]) * float(c["k_pages"][p, 0, j, d]) for d in range(16)) / 4 for p, j in rows]
            z = sum(math.exp(v) for v in s)
            assert abs(math.log(z) - float(lse[0, h, i])) < 1e-5
            for d in (0, 7):
                want = sum(math.exp(v) / z * float(c["v_pages"][p, 0, j, d]) for v, (p, j) in zip(s, rows))
                assert abs(want - float(o[0, i, h, d])) < 1e-5
    assert abs(float(c["weight"].sum()) - 4) < 1e-9  # four rows' weights


def _c_cache(nat, **over):
    a = dict(num_pages=8, kv_heads=2, page_size=16, head_dim=64, batch=2, pages_per_seq=4, k_pages=4096, v_pages=4096,
             ks=(2048, 1024, 64), vs=(2048, 1024, 64), page_table=4096, table_stride=4, lengths=4096, seen=4096, weight=4096,
             position=4096)
    a.update(over)
    return nat.KvCache(a["num_pages"], a["kv_heads"], a["page_size"], a["head_dim"], a["batch"], a["pages_per_seq"], a["k_pages"],
                       a["v_pages"], (ctypes.c_int64 * 3)(*a["ks"]), (ctypes.c_int64 * 3)(*a["vs"]), a["page_table"],
                       a["table_stride"], a["lengths"], a["seen"], a["weight"], a["position"])


BAD_CACHES = [
    (dict(head_dim=96), 2, "head dim"),
    (dict(page_size=24), 2, "multiple of 16"),
    (dict(page_size=0), 2, "multiple of 16"),
    (dict(num_pages=0), 1, "sizes"),
    (dict(batch=-1), 1, "sizes"),
    (dict(batch=70000), 2, "too large"),
    (dict(pages_per_seq=1 << 26), 2, "too large"),
    (dict(k_pages=0), 1, "null"),
    (dict(v_pages=4100), 1, "aligned"),
    (dict(ks=(2048, 1024, 60)), 1, "multiples of 8"),
    (dict(vs=(2048, 0, 64)), 1, "multiples of 8"),
    (dict(ks=(2048, 1024, 1 << 26)), 2, "slot"),
    (dict(lengths=0), 1, "lengths"),
    (dict(page_table=0), 1, "page_table"),
    (dict(table_stride=3), 1, "overlap"),
    (dict(weight=0), 1, "both"),
    (dict(weight=4104), 1, "aligned"),
    (dict(position=4100), 1, "aligned"),
]


@pytest.mark.parametrize("over,code,needle", BAD_CACHES)
def test_c_entries_reject_bad_caches(over, code, needle):
    from dmad_amd import _native as nat

    lib, p = nat.lib(), ctypes.c_void_p
    c = ctypes.byref(_c_cache(nat, **over))
    n = ctypes.c_size_t(0)
    s = (ctypes.c_int64 * 4)(256, 128, 64, 1)
    calls = [
        lambda: lib.dmad_paged_attn_workspace_bytes(c, 1, 4, 1, ctypes.byref(n)),
        lambda: lib.dmad_paged_attn(0, c, 1, 4, p(256), s, 0, 0, 0.125, p(256), p(256), p(256), 1 << 40, p(0)),
        lambda: lib.dmad_kv_evict_workspace_bytes(c, 8, ctypes.byref(n)),
        lambda: lib.dmad_kv_evict(0, c, 8, 0, 0, p(256), 1 << 40, p(0)),
        lambda: lib.dmad_qk_norm_rope_append(0, 0, 1, 4, p(256), p(256), p(256), s, s, s, p(0), p(0), p(0), 0, 0.0, p(256), c, p(0)),
    ]
    for call in calls:
        assert call() == code
        assert needle in lib.dmad_last_error().decode()


def test_c_entries_reject_bad_arguments():
    from dmad_amd import _native as nat

    lib, p = nat.lib(), ctypes.c_void_p
    c, bare = ctypes.byref(_c_cache(nat)), ctypes.byref(_c_cache(nat, weight=0, position=0))
    s = (ctypes.c_int64 * 4)(256, 128, 64, 1)

    def attn(cache=c, dtype=0, S=1, Hq=4, q=256, acc=0, scale=0.125, o=256, ws=256, size=1 << 40, strides=s):
        return lib.dmad_paged_attn(dtype, cache, S, Hq, p(q), strides, 0, acc, scale, p(o), p(256), p(ws), size, p(0))

    assert attn(cache=None) == 1
    assert attn(dtype=2) == 2 and attn(dtype=5) == 2
    assert attn(Hq=3) == 1 and attn(Hq=0) == 1 and attn(S=-1) == 1
    assert attn(q=0) == 1 and attn(q=264) == 1 and attn(o=0) == 1 and attn(o=8) == 1
    assert attn(scale=0.0) == 2 and attn(scale=-1.0) == 2 and attn(scale=math.nan) == 2
    # finite in 64 bits, not in 32; and so near the largest that log2(e) times it is not
    assert attn(scale=1e39) == 2 and attn(scale=3e38) == 2 and attn(scale=1e-50) == 2
    assert attn(cache=bare, acc=1) == 1
    assert attn(acc=1, ws=0) == 3 and attn(acc=1, size=64) == 3 and attn(acc=1, ws=272) == 3
    assert attn(S=1 << 28, Hq=64) == 2
    assert attn(S=0) == 0

    def evict(cache=c, keep=8, recent=0, sink=0, ws=256, size=1 << 40):
        return lib.dmad_kv_evict(0, cache, keep, recent, sink, p(ws), size, p(0))

    assert evict(cache=bare) == 1 and evict(keep=0) == 1 and evict(recent=-1) == 1 and evict(sink=-1) == 1
    assert evict(recent=9) == 1 and evict(recent=5, sink=4) == 1 and evict(recent=1 << 62, sink=1 << 62) == 1
    assert evict(ws=0) == 3 and evict(size=8) == 3
    assert evict(keep=64) == 0  # nothing can be longer

    def app(cache=c, S=1, Hq=4, q=256, k=256, oq=256, f=0, rows=0, eps=0.0, wd=0):
        return lib.dmad_qk_norm_rope_append(0, wd, S, Hq, p(q), p(k), p(256), s, s, s, p(0), p(0), p(f), rows, eps, p(oq), cache, p(0))

    assert app(q=0) == 1 and app(k=0) == 1 and app(oq=0) == 1 and app(Hq=0) == 1 and app(f=256, rows=0) == 1
    assert app(eps=-1.0) == 1 and app(wd=1) == 2 and app(S=0) == 0


def test_calls_off_the_gpu_raise():
    from dmad_amd import PagedKVCache

    with pytest.raises(RuntimeError, match="GPU only"):
        PagedKVCache.allocate(1, 16, 1, 16, device="cpu")


# ---------------------------------------------------------------- on the GPU


def _make(dev, B, Hk, D, dtype, page, lengths, room=0, extra=2, nhd=False, seed=0, weights=True, seen_ahead=0):
    """A cache of mixed pages holding `lengths` slots; everything else in the pool is NaN."""
    from dmad_amd import PagedKVCache

    g = torch.Generator().manual_seed(seed)
    M = max(1, -(-(max(lengths) + room) // page))
    N = B * M + extra
    table = torch.randperm(N, generator=g)[:B * M].view(B, M).to(torch.int32)
    shape = (N, page, Hk, D) if nhd else (N, Hk, page, D)
    c = dict(k_pages=torch.full(shape, math.nan, dtype=dtype), v_pages=torch.full(shape, math.nan, dtype=dtype),
             weight=torch.full((N, Hk, page), math.nan), position=torch.full((N, Hk, page), -1, dtype=torch.int32))
    if nhd:
        c["k_pages"], c["v_pages"] = c["k_pages"].transpose(1, 2), c["v_pages"].transpose(1, 2)
    for b, n in enumerate(lengths):
        k, v = (torch.randn(n, Hk, D, generator=g) * sd for sd in (1.5, 1.0))
        w = torch.rand(n, Hk, generator=g) ** 4
        w[torch.rand(n, Hk, generator=g) < 0.2] = 0.0
        for j in range(-(-n // page)):
            m = min(page, n - j * page)
            rows = slice(j * page, j * page + m)
            at = int(table[b, j])
            c["k_pages"][at, :, :m] = k[rows].transpose(0, 1).to(dtype)
            c["v_pages"][at, :, :m] = v[rows].transpose(0, 1).to(dtype)
            c["weight"][at, :, :m] = w[rows].t()
            c["position"][at, :, :m] = torch.arange(rows.start, rows.stop, dtype=torch.int32)
    lens = torch.tensor(lengths, dtype=torch.int32)

    def up(t):
        return torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=dev).copy_(t)

    return PagedKVCache(up(c["k_pages"]), up(c["v_pages"]), table.to(dev), lens.to(dev), (lens + seen_ahead).to(dev),
                        up(c["weight"]) if weights else None, up(c["position"]) if weights else None)


def _same(name, a, b):
    """Equal, NaN to NaN."""
    a, b = a.cpu().float(), b.cpu().float()
    assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a.nan_to_num(0.0), b.nan_to_num(0.0)), name


def _check_attention(got, ref, dtype, D, accumulated=None, before=None):
    o, lse = got
    ro, rlse, (pv, sv, size) = ref
    u = torch.finfo(dtype).eps / 2
    es = (D + 8) * F32 * size + 64 * F32 * (1 + rlse.transpose(1, 2)[..., None].abs().nan_to_num(0, posinf=0))
    tol = (u * (1 + 1e-3) + 2 * es) * pv + u * (1 + 1e-3) * ro.abs() + 1e-30
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25 * (sv + 1)
    err = (o.cpu().double() - ro).abs()
    assert torch.isfinite(o).all()
    print(f"  o: {float((err / tol).max()):.2f} of its bound", flush=True)
    assert (err <= tol).all()
    none = torch.isinf(rlse)
    assert torch.equal(lse.cpu() == -math.inf, none)
    err = (lse.cpu().double() - rlse).abs()[~none]
    assert (err <= es.amax(-1).transpose(1, 2)[~none]).all()


ATTEND = [
    # B, S, Hq, Hk, D, dtype, page, lengths, causal, accumulate
    (1, 1, 1, 1, 128, "bf16", 16, [1], False, True),
    (2, 1, 2, 2, 64, "fp16", 16, [0, 16], False, True),
    (3, 1, 4, 1, 128, "bf16", 16, [17, 31, 33], False, True),
    (1, 1, 12, 12, 64, "fp16", 16, [257], False, False),
    (2, 1, 8, 2, 16, "bf16", 32, [127, 129], False, True),
    (2, 2, 6, 3, 32, "fp16", 48, [500, 95], True, True),
    (1, 4, 64, 8, 128, "bf16", 64, [1000], True, True),
    (2, 7, 24, 8, 128, "fp16", 16, [300, 3], True, True),
    (1, 1, 5, 5, 256, "bf16", 16, [700], False, True),
    (2, 5, 10, 2, 256, "fp16", 64, [130, 4], True, False),
    (1, 40, 2, 1, 64, "bf16", 128, [390], True, True),
    (1, 33, 3, 3, 128, "bf16", 16, [33], True, False),
    (70, 1, 2, 1, 64, "bf16", 16, [(7 * i) % 61 for i in range(70)], False, True),
    (1, 1, 2, 2, 128, "bf16", 16, [9001], False, True),
    (3, 3, 16, 1, 32, "bf16", 16, [2, 1500, 640], True, True),
    (2, 1, 1, 1, 16, "bf16", 16, [9000, 700], False, True),
    (130, 1, 1, 1, 16, "fp16", 16, [(37 * i) % 400 for i in range(130)], False, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,S,Hq,Hk,D,dtype,page,lengths,causal,accumulate", ATTEND)
def test_attention(gpu, B, S, Hq, Hk, D, dtype, page, lengths, causal, accumulate):
    from dmad_amd import paged_attention

    print(f"case attend B={B} S={S} Hq={Hq} Hk={Hk} D={D} {dtype} page={page} lengths={lengths[:4]} causal={causal}", flush=True)
    t = DTYPES[dtype]
    cache = _make(gpu, B, Hk, D, t, page, lengths, room=5, seed=D + S, nhd=page == 48)
    q = (torch.randn(B, S, Hq, D, generator=torch.Generator().manual_seed(1)) * 1.5).to(t)
    c = st.cache_of(cache)
    ref = st.attend(c, q, causal=causal, accumulate=accumulate)
    before = cache.weight.clone()
    got = paged_attention(q.to(gpu), cache, causal=causal, accumulate=accumulate, return_lse=True)
    torch.cuda.synchronize()
    _check_attention(got, ref, t, D)
    if accumulate:
        w, r = cache.weight.cpu().double(), c["weight"].double()
        _same("weights of unused slots", torch.isnan(w).float(), torch.isnan(r).float())
        share = (r - before.cpu().double()).nan_to_num(0)
        # each p is off by the factor of its score and lse, the sum by float32's steps
        worst = float(ref[2][2].max()) * (D + 8) * F32 * 2 + 128 * F32 * (1 + float(ref[1][~torch.isinf(ref[1])].abs().max()) if (~torch.isinf(ref[1])).any() else 1)
        assert ((w - r).abs().nan_to_num(0) <= worst * share + 2 * F32 * r.abs().nan_to_num(0) + 1e-30).all()
    else:
        _same("weights", cache.weight, before)
    # the same again bit for bit, and without lse
    again = paged_attention(q.to(gpu), cache, causal=causal)
    assert torch.equal(again, got[0])


@pytest.mark.gpu
def test_attention_of_missing_pages_and_odd_lengths(gpu):
    """Ids outside the pool hide their slots; lengths beyond the table or negative are clipped; a sequence
    without a readable slot gives zeros and -inf."""
    from dmad_amd import paged_attention

    cache = _make(gpu, 6, 2, 64, torch.bfloat16, 16, [100, 100, 100, 100, 100, 100], seed=3)
    N = cache.k_pages.shape[0]
    cache.page_table[0, 0] = -1
    cache.page_table[1, 3] = N
    cache.page_table[1, 6] = 2 ** 31 - 1
    cache.page_table[2, :] = -(2 ** 31)
    cache.lengths[3] = -5
    cache.lengths[4] = 0
    cache.page_table[5, 1:5] = -1
    q = torch.randn(6, 2, 4, 64, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    for causal in (False, True):
        c = st.cache_of(cache)
        ref = st.attend(c, q, causal=causal, accumulate=True)
        w = cache.weight.clone()
        got = paged_attention(q.to(gpu), cache, causal=causal, accumulate=True, return_lse=True)
        torch.cuda.synchronize()
        _check_attention(got, ref, torch.bfloat16, 64)
        assert torch.equal(got[0][2:5], torch.zeros_like(got[0][2:5])) and torch.isneginf(got[1][2:5]).all()
        assert torch.allclose(cache.weight.cpu().double(), c["weight"].double(), rtol=1e-4, atol=1e-6, equal_nan=True)
        cache.weight.copy_(w)
    # a length beyond the table: all its slots, the NaN ones beyond the data among them, reach that sequence alone
    cache.lengths[4] = 10 ** 9
    o = paged_attention(q.to(gpu), cache)
    assert torch.isnan(o[4]).all() and torch.isfinite(o[:4]).all() and torch.isfinite(o[5]).all()


@pytest.mark.gpu
def test_attention_scores_of_any_size(gpu):
    """Scores far apart and all very low keep their softmax; an infinite or NaN key or value reaches its own
    sequence and key head and no other."""
    from dmad_amd import paged_attention

    for dtype in (torch.bfloat16, torch.float16):
        cache = _make(gpu, 2, 2, 64, dtype, 16, [300, 260], seed=4)
        c = st.cache_of(cache)
        q = torch.randn(2, 1, 4, 64, generator=torch.Generator().manual_seed(5)).to(dtype)
        for scale in (1e-3, 1.0, 30.0):
            ref = st.attend(c, q, scale=scale)
            got = paged_attention(q.to(gpu), cache, sm_scale=scale, return_lse=True)
            _check_attention(got, ref, dtype, 64)
        low = torch.full((2, 1, 4, 64), -200.0).to(dtype)
        page, slot = st.locate(c, 0, 290)
        cache.k_pages[cache.page_table[0].long()] = 200.0
        c = st.cache_of(cache)
        _check_attention(paged_attention(low.to(gpu), cache, return_lse=True), st.attend(c, low), dtype, 64)
        clean = paged_attention(q.to(gpu), cache)
        for where, value in (("k_pages", math.nan), ("v_pages", math.inf), ("v_pages", math.nan)):
            keep = getattr(cache, where)[page, 1, slot].clone()
            getattr(cache, where)[page, 1, slot] = value
            o = paged_attention(q.to(gpu), cache)
            assert not torch.isfinite(o[0, 0, 2:]).any(), where
            assert torch.equal(o[0, 0, :2], clean[0, 0, :2]) and torch.equal(o[1], clean[1])
            getattr(cache, where)[page, 1, slot] = keep


@pytest.mark.gpu
@pytest.mark.parametrize("D,S,Hq,dtype", [(64, 4, 8, "bf16"), (16, 3, 2, "fp16"), (128, 9, 8, "bf16"), (256, 2, 2, "fp16"), (32, 40, 2, "bf16")])
def test_hidden_tokens_do_not_reach_earlier_ones(gpu, D, S, Hq, dtype):
    """With causal, whatever the values (and keys) of later new tokens hold: a token that does not see them is as
    if they were not there, one that sees an infinity or NaN is not finite."""
    from dmad_amd import paged_attention

    t = DTYPES[dtype]
    for length in (S, 37 + S, 300 + S):
        cache = _make(gpu, 1, 2, D, t, 16, [length], seed=D + length)
        q = torch.randn(1, S, Hq, D, generator=torch.Generator().manual_seed(3)).to(t)
        clean = paged_attention(q.to(gpu), cache, causal=True, return_lse=True)
        _check_attention(clean, st.attend(st.cache_of(cache), q, causal=True), t, D)
        for token in {1, S - 1}:
            page, slot = st.locate(st.cache_of(cache), 0, length - S + token)
            for name, value in (("v_pages", math.inf), ("v_pages", math.nan), ("k_pages", math.nan)):
                pages = getattr(cache, name)
                keep = pages[page, 0, slot].clone()
                pages[page, 0, slot] = value
                o = paged_attention(q.to(gpu), cache, causal=True)
                half = Hq // 2  # the query heads of key head 0
                assert torch.equal(o[:, :token], clean[0][:, :token]), (length, token, name)
                assert torch.equal(o[:, :, half:], clean[0][:, :, half:]), (length, token, name)
                assert not torch.isfinite(o[:, token:, :half]).any(), (length, token, name)
                pages[page, 0, slot] = keep


@pytest.mark.gpu
def test_attention_reads_strided_queries(gpu):
    """Queries as a slice of a projection's output, as a transpose and unaligned; keys in [N, P, H, D] storage."""
    from dmad_amd import paged_attention

    cache = _make(gpu, 2, 2, 64, torch.bfloat16, 32, [70, 200], seed=21, nhd=True)
    g = torch.Generator().manual_seed(22)
    qkv = torch.randn(2, 3, 8, 64, generator=g).to(torch.bfloat16).to(gpu)
    want = paged_attention(qkv[:, :, :4].contiguous(), cache, causal=True)
    assert torch.equal(paged_attention(qkv[:, :, :4], cache, causal=True), want)
    assert torch.equal(paged_attention(qkv[:, :, :4].transpose(1, 2).contiguous().transpose(1, 2), cache, causal=True), want)
    flat = torch.zeros(2 * 3 * 4 * 64 + 1, device=gpu, dtype=torch.bfloat16)
    flat[1:] = qkv[:, :, :4].reshape(-1)
    assert torch.equal(paged_attention(flat[1:].view(2, 3, 4, 64), cache, causal=True), want)
    one = qkv[:, :1, :4].expand(2, 3, 4, 64)
    assert torch.equal(paged_attention(one, cache), paged_attention(one.contiguous(), cache))


@pytest.mark.gpu
def test_shared_pages_on_two_streams(gpu):
    """Sequences that begin with the same pages, read by two calls at once on two streams and by one after
    another: the same results, those of sequences with pages of their own."""
    from dmad_amd import PagedKVCache, paged_attention

    Hq, Hk, D, dtype = 8, 2, 128, torch.bfloat16
    lengths = [700, 640, 1300, 16]
    own = _make(gpu, 4, Hk, D, dtype, 16, lengths, seed=50)
    table = own.page_table.clone()
    table[1:3, :40] = table[0, :40]  # 640 slots in common
    shared = PagedKVCache(own.k_pages, own.v_pages, table, own.lengths, own.seen)
    g = torch.Generator().manual_seed(51)
    qs = [torch.randn(4, S, Hq, D, generator=g).to(dtype) for S in (1, 3)]
    calls = [dict(causal=False), dict(causal=True)]
    dev = [q.to(gpu) for q in qs]
    want = []
    for q, x, kw in zip(qs, dev, calls):
        want.append(paged_attention(x, shared, return_lse=True, **kw))
        torch.cuda.synchronize()
        _check_attention(want[-1], st.attend(st.cache_of(shared), q, causal=kw["causal"]), dtype, D)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(paged_attention(dev[i], shared, return_lse=True, **calls[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for o, lse in got[i]:
            assert torch.equal(o, want[i][0]) and torch.equal(lse, want[i][1])


@pytest.mark.gpu
def test_attention_equals_the_dense_one(gpu):
    """Against the package's own dense attention over the same keys."""
    from dmad_amd import paged_attention, plain_attention

    cache = _make(gpu, 1, 8, 128, torch.bfloat16, 16, [4000], seed=6)
    q = torch.randn(1, 16, 8, 128, generator=torch.Generator().manual_seed(7)).to(torch.bfloat16).to(gpu)
    used = cache.page_table[0].long()
    k, v = (p[used].transpose(0, 1).reshape(1, 8, -1, 128)[:, :, :4000].contiguous() for p in (cache.k_pages, cache.v_pages))
    dense = plain_attention(q.transpose(1, 2), k, v).transpose(1, 2).float()
    o = paged_attention(q, cache).float()
    assert float((o - dense).norm() / dense.norm()) < 5e-3


APPEND = [
    # B, S, Hq, Hk, D, dtype, page, lengths, weights' type
    (1, 1, 1, 1, 16, "bf16", 16, [0], "bf16"),
    (3, 1, 8, 2, 128, "bf16", 16, [15, 16, 0], "fp32"),
    (2, 5, 6, 3, 64, "fp16", 48, [46, 100], "fp16"),
    (1, 130, 40, 40, 128, "bf16", 64, [61], "bf16"),
    (2, 3, 9, 1, 32, "fp16", 16, [0, 31], "fp32"),
    (2, 2, 4, 4, 256, "bf16", 32, [31, 64], "bf16"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,S,Hq,Hk,D,dtype,page,lengths,wtype", APPEND)
def test_append(gpu, B, S, Hq, Hk, D, dtype, page, lengths, wtype):
    from dmad_amd import qk_norm_rope_append
    from test_qk_norm_rope import _check, _pair_size

    print(f"case append B={B} S={S} Hq={Hq} Hk={Hk} D={D} {dtype} page={page} lengths={lengths}", flush=True)
    t = DTYPES[dtype]
    cache = _make(gpu, B, Hk, D, t, page, lengths, room=S, seed=D, nhd=page == 48, seen_ahead=3)
    g = torch.Generator().manual_seed(8)
    qkv = torch.randn(B, S, Hq + 2 * Hk, D, generator=g).to(t)
    wq, wk = ((1 + 0.2 * torch.randn(D, generator=g)).to({"fp32": torch.float32, **DTYPES}[wtype]) for _ in range(2))
    freqs = torch.rand(max(lengths) + 3 + S, D // 2, generator=g) * 300
    c, before = st.cache_of(cache), st.cache_of(cache)
    q, k, v = qkv.split((Hq, Hk, Hk), dim=2)
    rq, rk = st.append(c, q, k, v, wq, wk, 1e-6, freqs)
    dq, dk, dv = qkv.to(gpu).split((Hq, Hk, Hk), dim=2)
    got = qk_norm_rope_append(dq, dk, dv, wq.to(gpu), wk.to(gpu), 1e-6, freqs.to(gpu), cache)
    torch.cuda.synchronize()
    _check("q", got, rq, _pair_size(rq))
    after = st.cache_of(cache)
    for b in range(B):
        for i in range(S):
            at = st.locate(c, b, lengths[b] + i)
            _check(f"k {b} {i}", after["k_pages"][at[0], :, at[1]], rk[b, i], _pair_size(rk[b, i]))
            before["k_pages"][at[0], :, at[1]] = after["k_pages"][at[0], :, at[1]]
    _same("other slots", after["k_pages"], before["k_pages"])
    for n in ("v_pages", "weight", "position", "lengths", "seen"):
        _same(n, after[n], c[n])


@pytest.mark.gpu
def test_append_where_there_is_no_room(gpu):
    """Tokens beyond the capacity or on missing pages are dropped, positions beyond the angles give NaN, and
    keys appended as they are keep their bits."""
    from dmad_amd import append_kv, qk_norm_rope_append

    cache = _make(gpu, 4, 2, 32, torch.bfloat16, 16, [30, 10, 32, 5], seed=9)
    cache.page_table[1, 0] = -1
    cache.lengths[3] = -7
    g = torch.Generator().manual_seed(10)
    k, v = (torch.randn(4, 5, 2, 32, generator=g).to(torch.bfloat16) for _ in range(2))
    k[0, 0, 0, 0] = math.inf
    c = st.cache_of(cache)
    st.append(c, None, k, v, None, None, 0.0, None)
    append_kv(k.to(gpu), v.to(gpu), cache)
    torch.cuda.synchronize()
    for n in st.FIELDS:
        _same(n, getattr(cache, n), c[n])
    assert cache.lengths.tolist() == [32, 15, 32, 5] and cache.seen.tolist() == [35, 15, 37, 10]
    # angles for positions 0..35 only
    cache.lengths.zero_()
    q = torch.randn(4, 2, 6, 32, generator=g).to(torch.bfloat16).to(gpu)
    w, f = torch.ones(32, device=gpu), torch.rand(36, 16, generator=g).to(gpu)
    got = qk_norm_rope_append(q, q[:, :, :2], q[:, :, 2:4], w, w, 1e-6, f, cache)
    bad = torch.tensor([[s + i >= 36 for i in range(2)] for s in (35, 15, 37, 10)])
    assert torch.equal(torch.isnan(got.float()).all(-1).all(-1).cpu(), bad)
    assert torch.equal(torch.isnan(got.float()).any(-1).any(-1).cpu(), bad)
    # negative counts have no angles either
    cache.seen.fill_(-2 ** 31)
    assert torch.isnan(qk_norm_rope_append(q, q[:, :, :2], q[:, :, 2:4], w, w, 1e-6, f, cache).float()).all()


EVICT = [
    # B, Hk, D, dtype, page, lengths, keep, recent, sink
    (1, 1, 16, "bf16", 16, [2], 1, 0, 0),
    (2, 2, 64, "fp16", 16, [33, 32], 32, 4, 1),
    (3, 1, 128, "bf16", 16, [0, 100, 64], 64, 16, 4),
    (2, 3, 32, "bf16", 48, [500, 333], 100, 0, 0),
    (1, 2, 256, "fp16", 64, [1100], 1000, 100, 0),
    (2, 2, 64, "bf16", 16, [2500, 90], 77, 30, 47),
    (1, 1, 64, "bf16", 16, [5000], 4999, 0, 3),
    (1, 2, 16, "bf16", 128, [36000], 20001, 77, 0),
    (2, 1, 16, "bf16", 16, [4096, 4097], 4095, 0, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,Hk,D,dtype,page,lengths,keep,recent,sink", EVICT)
def test_evict(gpu, B, Hk, D, dtype, page, lengths, keep, recent, sink):
    from dmad_amd import evict_low_weight

    print(f"case evict B={B} Hk={Hk} D={D} page={page} lengths={lengths} keep={keep} recent={recent} sink={sink}", flush=True)
    cache = _make(gpu, B, Hk, D, DTYPES[dtype], page, lengths, room=7, seed=keep, nhd=page == 48)
    for again in range(2):  # a second cut finds slots out of order
        c = st.cache_of(cache)
        k = keep if again == 0 else max(1, keep // 2)
        r, s = (recent, sink) if again == 0 else (recent // 2, sink // 2)
        st.evict(c, k, r, s)
        evict_low_weight(cache, k, recent=r, sink=s)
        torch.cuda.synchronize()
        for n in st.FIELDS:
            _same(n, getattr(cache, n), c[n])


@pytest.mark.gpu
@pytest.mark.parametrize("size", [300, 5000, 33100])
@pytest.mark.parametrize("kind", ["equal", "zeros of both signs", "infinities and NaN", "all recent", "negative", "missing pages"])
def test_evict_order(gpu, kind, size):
    """Ties, signs and what is not a number, for keys in a little and in much LDS and in memory."""
    from dmad_amd import evict_low_weight

    print(f"case evict order {kind} {size}", flush=True)
    cache = _make(gpu, 2, 1, 16, torch.bfloat16, 16, [size, 211], seed=11)
    g = torch.Generator().manual_seed(12)
    w = torch.rand(cache.weight.shape, generator=g)
    if kind == "equal":
        w = torch.ones_like(w)
    elif kind == "zeros of both signs":
        w = torch.where(w < 0.5, torch.tensor(-0.0), torch.tensor(0.0))
    elif kind == "infinities and NaN":
        w = torch.where(w < 0.1, torch.tensor(math.nan), torch.where(w < 0.4, torch.tensor(math.inf), torch.where(w < 0.7, torch.tensor(-math.inf), w)))
    elif kind == "negative":
        w = w - 0.7
    elif kind == "all recent":
        cache.position.fill_(10 ** 6)
    cache.weight.copy_(w)
    if kind == "missing pages":
        cache.page_table[0, 2] = -1
        cache.page_table[0, 15] = cache.k_pages.shape[0]
        cache.page_table[1, 12] = -9
    c = st.cache_of(cache)
    keep = 128 if size < 1000 else size // 2 + 9
    st.evict(c, keep, 16, 4)
    evict_low_weight(cache, keep, recent=16, sink=4)
    torch.cuda.synchronize()
    for n in st.FIELDS:
        _same(n, getattr(cache, n), c[n])


@pytest.mark.gpu
def test_offsets_beyond_32_bits(gpu):
    """A pool of 5 GiB per side, a few pages at its end."""
    from dmad_amd import PagedKVCache, evict_low_weight, paged_attention, qk_norm_rope_append

    N, Hk, P, D = 5 * 2 ** 30 // (8 * 64 * 128 * 2), 8, 64, 128
    k_pages = torch.empty((N, Hk, P, D), device=gpu, dtype=torch.bfloat16)
    v_pages = torch.empty_like(k_pages)
    table = torch.tensor([[N - 1, N - 3], [N - 2, 0]], device=gpu, dtype=torch.int32)
    small = table.long().view(-1)
    g = torch.Generator(device=gpu).manual_seed(0)
    for pages in (k_pages, v_pages):
        pages[small] = torch.randn((4, Hk, P, D), generator=g, device=gpu).to(torch.bfloat16)
    lens = torch.tensor([100, 64], device=gpu, dtype=torch.int32)
    weight = torch.rand((N, Hk, P), generator=g, device=gpu)
    position = torch.arange(P, device=gpu, dtype=torch.int32).expand(N, Hk, P).contiguous()
    big = PagedKVCache(k_pages, v_pages, table, lens, lens.clone(), weight, position)
    ids = torch.arange(4, device=gpu, dtype=torch.int32).view(2, 2)
    little = PagedKVCache(k_pages[small].clone(), v_pages[small].clone(), ids, lens.clone(), lens.clone(), weight[small].clone(),
                          position[small].clone())
    q = torch.randn((2, 1, 16, D), generator=g, device=gpu).to(torch.bfloat16)
    kv = torch.randn((2, 1, Hk, D), generator=g, device=gpu).to(torch.bfloat16)
    w, f = torch.ones(D, device=gpu), torch.rand((200, D // 2), generator=g, device=gpu)
    outs = []
    for cache in (big, little):
        a = qk_norm_rope_append(q, kv, kv, w, w, 1e-6, f, cache)
        o = paged_attention(a, cache, accumulate=True)
        evict_low_weight(cache, 60, recent=3)
        outs.append((a, o, paged_attention(a, cache)))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    for n in ("k_pages", "v_pages", "weight", "position"):
        assert torch.equal(getattr(big, n)[small], getattr(little, n)), n


def _decode(cache, steps, wq, wk, freqs, keep):
    from dmad_amd import evict_low_weight, paged_attention, qk_norm_rope_append

    outs = []
    for q, k, v in steps:
        q = qk_norm_rope_append(q, k, v, wq, wk, 1e-6, freqs, cache)
        outs.append(paged_attention(q, cache, causal=True, accumulate=True))
        evict_low_weight(cache, keep, recent=8, sink=2)
    return outs


def _steps(dev, B, Hq, Hk, D, dtype, sizes, seed):
    g = torch.Generator().manual_seed(seed)
    return [[torch.randn(B, S, h, D, generator=g).to(dtype).to(dev) for h in (Hq, Hk, Hk)] for S in sizes]


@pytest.mark.gpu
def test_decoding_with_eviction(gpu):
    """A prompt, then tokens one, three and one at a time against a cache that is cut to 40 slots after every
    step, each call against the oracle on a copy of the cache it found. Slots and positions agree in every step."""
    from dmad_amd import PagedKVCache

    B, Hq, Hk, D, dtype = 2, 8, 2, 64, torch.bfloat16
    cache = PagedKVCache.allocate(B, 80, Hk, D, dtype, gpu, page_size=16)
    assert cache.capacity == 80
    g = torch.Generator().manual_seed(20)
    wq, wk = ((1 + 0.2 * torch.randn(D, generator=g)).to(dtype) for _ in range(2))
    freqs = torch.rand(200, D // 2, generator=g) * 50
    total = 0
    for n, (q, k, v) in enumerate(_steps(gpu, B, Hq, Hk, D, dtype, [37, 1, 3, 1, 1, 8, 1], 21)):
        from dmad_amd import evict_low_weight, paged_attention, qk_norm_rope_append

        c = st.cache_of(cache)
        st.append(c, q.cpu(), k.cpu(), v.cpu(), wq, wk, 1e-6, freqs)
        qn = qk_norm_rope_append(q, k, v, wq.to(gpu), wk.to(gpu), 1e-6, freqs.to(gpu), cache)
        total += q.shape[1]
        assert cache.lengths.tolist() == c["lengths"].tolist() and cache.seen.tolist() == [total] * B
        c = st.cache_of(cache)
        ref = st.attend(c, qn.cpu(), causal=True, accumulate=True)
        got = paged_attention(qn, cache, causal=True, accumulate=True, return_lse=True)
        _check_attention(got, ref, dtype, D)
        c = st.cache_of(cache)
        st.evict(c, 40, 8, 2)
        evict_low_weight(cache, 40, recent=8, sink=2)
        for name in st.FIELDS:
            _same(f"{name} after step {n}", getattr(cache, name)[:] if name != "lengths" else cache.lengths, c[name])
        for h in range(Hk):  # positions of the slots in use are distinct, the last ones and the sinks among them
            at = [int(cache.position[p, h, s]) for p, s in (st.locate(c, 0, j) for j in range(int(cache.lengths[0])))]
            assert len(set(at)) == len(at) and {0, 1, *range(max(0, total - 8), total)} <= set(at)


@pytest.mark.gpu
def test_captured_steps_follow_the_cache(gpu):
    """One captured step replayed token by token: lengths, pages and evictions are the device's, so every
    replay is the eager step that stands there. Two graphs of the same calls do not disturb each other."""
    from dmad_amd import PagedKVCache

    B, Hq, Hk, D, dtype = 3, 8, 2, 128, torch.bfloat16
    g = torch.Generator().manual_seed(30)
    wq, wk = ((1 + 0.2 * torch.randn(D, generator=g)).to(gpu) for _ in range(2))
    freqs = (torch.rand(600, D // 2, generator=g) * 50).to(gpu)
    steps = _steps(gpu, B, Hq, Hk, D, dtype, [1] * 6, 31)

    def fresh():
        cache = PagedKVCache.allocate(B, 400, Hk, D, dtype, gpu, page_size=16)
        _decode(cache, _steps(gpu, B, Hq, Hk, D, dtype, [300], 32), wq, wk, freqs, 301)
        cache.lengths[1] = 7
        return cache

    eager = fresh()
    want = [o.clone() for o in _decode(eager, steps, wq, wk, freqs, 300)]
    torch.cuda.synchronize()
    caches, graphs, ins, outs = [fresh() for _ in range(2)], [], [], []
    for cache in caches:
        saved = {n: getattr(cache, n).clone() for n in st.FIELDS}
        x = [t.clone() for t in steps[0]]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _decode(cache, [x], wq, wk, freqs, 300)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_decode(cache, [x], wq, wk, freqs, 300)[0])
        for n, t in saved.items():
            getattr(cache, n).copy_(t)
        graphs.append(graph)
        ins.append(x)
    for n, step in enumerate(steps):
        for i in range(2):
            for a, b in zip(ins[i], step):
                a.copy_(b)
            graphs[i].replay()
        junk = torch.randn(1024, 1024, device=gpu)
        (junk @ junk).sum().item()
        for i in range(2):
            assert torch.equal(outs[i], want[n]), (n, i)
    for cache in caches:
        for name in ("lengths", "seen"):
            assert torch.equal(getattr(cache, name), getattr(eager, name))


@pytest.mark.gpu
def test_refusals(gpu):
    from dmad_amd import PagedKVCache, append_kv, evict_low_weight, paged_attention, qk_norm_rope_append

    ok = PagedKVCache.allocate(2, 40, 2, 64, torch.bfloat16, gpu, page_size=16)
    assert ok.capacity == 48
    f = [getattr(ok, n) for n in ("k_pages", "v_pages", "page_table", "lengths", "seen", "weight", "position")]

    def built(**over):
        names = ("k_pages", "v_pages", "page_table", "lengths", "seen", "weight", "position")
        return PagedKVCache(**{**dict(zip(names, f)), **over})

    built()
    for error, over in [
        (ValueError, dict(v_pages=f[1][:1])),
        (ValueError, dict(k_pages=f[0][0])),
        (NotImplementedError, dict(v_pages=f[1].half())),
        (NotImplementedError, dict(k_pages=f[0].float(), v_pages=f[1].float())),
        (NotImplementedError, dict(k_pages=f[0][:, :, :8], v_pages=f[1][:, :, :8])),
        (NotImplementedError, dict(k_pages=f[0][..., :48], v_pages=f[1][..., :48])),
        (ValueError, dict(k_pages=f[0].transpose(2, 3).contiguous().transpose(2, 3))),
        (ValueError, dict(k_pages=f[0][:1].expand_as(f[0]))),
        (ValueError, dict(page_table=f[2].long())),
        (ValueError, dict(page_table=f[2].t())),
        (ValueError, dict(lengths=f[3][:1])),
        (ValueError, dict(seen=f[4].long())),
        (ValueError, dict(weight=None)),
        (ValueError, dict(weight=f[5].double())),
        (ValueError, dict(position=f[6][:, :1])),
        (ValueError, dict(weight=torch.zeros(f[5].numel() + 1, device=gpu)[1:].view(f[5].shape))),
        (RuntimeError, dict(lengths=f[3].cpu())),
    ]:
        with pytest.raises(error):
            built(**over)
    with pytest.raises(AttributeError, match="in place"):
        ok.lengths = f[3]
    with pytest.raises(NotImplementedError, match="multiple of 16"):
        PagedKVCache.allocate(1, 10, 1, 64, device=gpu, page_size=20)
    with pytest.raises(ValueError):
        PagedKVCache.allocate(0, 10, 1, 64, device=gpu)

    q, k = torch.zeros(2, 1, 4, 64, device=gpu, dtype=torch.bfloat16), torch.zeros(2, 1, 2, 64, device=gpu, dtype=torch.bfloat16)
    w = torch.ones(64, device=gpu)
    bare = built(weight=None, position=None)
    for error, call in [
        (TypeError, lambda: paged_attention(q, f[0])),
        (ValueError, lambda: paged_attention(q[:1], ok)),
        (ValueError, lambda: paged_attention(q[0], ok)),
        (ValueError, lambda: paged_attention(q[..., :32], ok)),
        (ValueError, lambda: paged_attention(q[:, :, :3], ok)),
        (ValueError, lambda: paged_attention(q.half(), ok)),
        (RuntimeError, lambda: paged_attention(q.cpu(), ok)),
        (NotImplementedError, lambda: paged_attention(q, ok, sm_scale=0.0)),
        (NotImplementedError, lambda: paged_attention(q, ok, sm_scale=math.nan)),
        (NotImplementedError, lambda: paged_attention(q, ok, sm_scale=1e39)),
        (ValueError, lambda: paged_attention(q, bare, accumulate=True)),
        (RuntimeError, lambda: paged_attention(q.clone().requires_grad_(True), ok)),
        (ValueError, lambda: append_kv(k, None, ok)),
        (ValueError, lambda: append_kv(k, q, ok)),
        (ValueError, lambda: append_kv(k, k.half(), ok)),
        (ValueError, lambda: append_kv(k, torch.cat((k, k), 1), ok)),
        (TypeError, lambda: append_kv(k, k, None)),
        (ValueError, lambda: qk_norm_rope_append(q, k, k, w, w, -1.0, None, ok)),
        (ValueError, lambda: qk_norm_rope_append(q, k, k, w[:32], w, 1e-6, None, ok)),
        (ValueError, lambda: qk_norm_rope_append(None, k, k, w, w, 1e-6, None, ok)),
        (ValueError, lambda: qk_norm_rope_append(q, k, k, w, w, 1e-6, torch.zeros(5, 64, device=gpu), ok)),
        (RuntimeError, lambda: qk_norm_rope_append(q, k, k, w.clone().requires_grad_(True), w, 1e-6, None, ok)),
        (ValueError, lambda: evict_low_weight(bare, 8)),
        (TypeError, lambda: evict_low_weight(None, 8)),
        (ValueError, lambda: evict_low_weight(ok, 0)),
        (ValueError, lambda: evict_low_weight(ok, 8, recent=-1)),
        (ValueError, lambda: evict_low_weight(ok, 8, recent=5, sink=4)),
    ]:
        with pytest.raises(error):
            call()
    assert ok.lengths.tolist() == [0, 0]
    # without weights everything else works
    append_kv(k, k, bare)
    assert torch.equal(paged_attention(q, bare), torch.zeros_like(q)) and bare.lengths.tolist() == [1, 1]
    # no new tokens, no sequences
    assert paged_attention(q[:, :0], bare).shape == (2, 0, 4, 64)
    append_kv(k[:, :0], k[:, :0], bare)
    assert bare.lengths.tolist() == [1, 1]
    none = PagedKVCache(f[0], f[1], f[2][:0], f[3][:0], f[4][:0])
    assert paged_attention(q[:0], none).shape == (0, 1, 4, 64)
    append_kv(k[:0], k[:0], none)


# ---------------------------------------------------------------- windows: pages missing in front and between


def test_oracle_eviction_of_a_window_by_hand():
    """128 slots whose first 64 lie on dropped pages. 64 are there: cut to 64 nothing goes. Cut to 20 (a sink that
    is no longer there, the last 16 positions, the heaviest of the rest) the sequence ends behind its 20th slot."""
    def window():
        c = dict(k_pages=torch.arange(128.0).view(8, 1, 16, 1).repeat(1, 1, 1, 16), v_pages=torch.zeros(8, 1, 16, 16),
                 page_table=torch.arange(8, dtype=torch.int32).view(1, 8).clone(), lengths=torch.tensor([128]),
                 seen=torch.tensor([128]), weight=torch.zeros(8, 1, 16), position=torch.arange(128).view(8, 1, 16).clone())
        c["page_table"][0, :4] = -1
        c["weight"].view(-1)[[70, 81, 90, 111]] = 2.0
        return c

    c, same = window(), window()
    st.evict(c, 64, recent=16)
    assert all(torch.equal(c[n], same[n]) for n in st.FIELDS)
    st.evict(c, 20, recent=16, sink=4)
    assert c["lengths"].tolist() == [84]
    live = [at for s in range(84) if (at := st.locate(c, 0, s)) is not None]
    held = [int(c["position"][p, 0, s]) for p, s in live]
    assert sorted(held) == [70, 81, 90, 111, *range(112, 128)]
    assert held[6] == 70 and held[17] == 81  # those that stay below the end have not moved
    assert [float(c["k_pages"][p, 0, s, 0]) for p, s in live] == held


WINDOW = [
    # capacity in pages, length, missing entries, keep, recent, sink
    (8, 128, [0, 1, 2, 3], 64, 16, 0),       # as many slots left as stay
    (8, 128, [0, 1, 2, 3], 65, 16, 4),       # fewer left than stay
    (8, 128, [0, 1, 2, 3], 48, 16, 0),
    (8, 128, [0, 1, 2, 3, 4, 5, 6, 7], 5, 2, 1),
    (8, 120, [0, 2, 5], 33, 8, 2),
    (8, 117, [6, 7], 20, 20, 0),             # the newest pages are the ones missing
    (40, 629, [*range(0, 20), 30], 100, 50, 3),
    (400, 6301, [*range(0, 250), 251, 260, 399], 1000, 128, 4),  # keys in much LDS
    (400, 6400, [*range(1, 398)], 20, 7, 9),
    (2200, 35000, [*range(0, 1500), 1700], 3000, 64, 0),  # keys in memory
]


@pytest.mark.gpu
@pytest.mark.parametrize("pages,length,missing,keep,recent,sink", WINDOW)
def test_evict_in_a_window(gpu, pages, length, missing, keep, recent, sink):
    """Missing pages hold nothing, so they do not use up `keep`: the newest and heaviest of the slots that are
    there stay, for a sequence beside one without missing pages."""
    from dmad_amd import evict_low_weight, paged_attention

    print(f"case evict window length={length} missing={len(missing)} keep={keep}", flush=True)
    cache = _make(gpu, 2, 2, 16, torch.bfloat16, 16, [length, max(1, length - 9)], room=16 * pages - length, seed=keep)
    assert cache.page_table.shape[1] == pages
    cache.page_table[0, missing] = -1
    for k, r, s in ((keep, recent, sink), (max(1, keep // 2), recent // 2, sink // 2)):
        c = st.cache_of(cache)
        there = [int(c["position"][p, 0, j]) for i in range(st.length(c, 0)) if (at := st.locate(c, 0, i)) for p, j in [at]]
        st.evict(c, k, r, s)
        evict_low_weight(cache, k, recent=r, sink=s)
        torch.cuda.synchronize()
        for n in st.FIELDS:
            _same(n, getattr(cache, n), c[n])
        live = [at for i in range(int(cache.lengths[0])) if (at := st.locate(c, 0, i)) is not None]
        assert len(live) == min(k, len(there))
        for h in range(2):
            held = {int(c["position"][p, h, j]) for p, j in live}
            assert held >= {t for t in there if t >= length - r or t < s}
    if there:
        assert torch.isfinite(paged_attention(torch.randn(2, 1, 2, 16, device=gpu).bfloat16(), cache, return_lse=True)[1]).all()


# ---------------------------------------------------------------- light slots beside a heavy one


LIGHT = [
    # D, S, Hq, dtype, length, binary orders that the light slots lie below the heavy one
    (64, 1, 1, "fp16", 3001, 16.7),
    (64, 1, 1, "fp16", 3001, 20.3),
    (128, 3, 2, "fp16", 2000, 18.5),
    (16, 1, 20, "fp16", 1500, 22.6),
    (256, 2, 1, "fp16", 900, 24.4),
    (32, 1, 1, "fp16", 40, 26.2),
    (64, 1, 1, "bf16", 3001, 20.3),
]


@pytest.mark.gpu
@pytest.mark.parametrize("D,S,Hq,dtype,length,orders", LIGHT)
def test_light_slots_keep_their_share(gpu, D, S, Hq, dtype, length, orders):
    """One heavy slot with zero values over a tail of equally light ones, which the output is made of. P enters its
    product rounded to the type, u of it each, whatever its size next to the heaviest: an absolute step that
    many equal slots share would add up. What is left of such a step is 2^-40 (2^-25 of half a subnormal step,
    2^-15 of the scaling) of sum |v| in fp16, and half a subnormal step of the output."""
    from dmad_amd import paged_attention

    print(f"case light D={D} S={S} Hq={Hq} {dtype} {length} {orders}", flush=True)
    t = DTYPES[dtype]
    cache = _make(gpu, 1, 1, D, t, 16, [length], seed=60)
    q = torch.zeros(1, S, Hq, D)
    q[..., 0] = 4.0
    c = st.cache_of(cache)
    for s in range(length):
        p, j = st.locate(c, 0, s)
        cache.k_pages[p, 0, j] = 0
        cache.v_pages[p, 0, j] = c["v_pages"][p, 0, j].abs()
    p, j = st.locate(c, 0, 5)
    cache.k_pages[p, 0, j, 0] = 8.0
    cache.v_pages[p, 0, j] = 0
    q, scale = q.to(t), orders * math.log(2) / 32
    o, lse = paged_attention(q.to(gpu), cache, sm_scale=scale, causal=True, return_lse=True)
    ro, rlse, (pv, sv, size) = st.attend(st.cache_of(cache), q, scale=scale, causal=True)
    u = torch.finfo(t).eps / 2
    es = (D + 8) * F32 * size + 64 * F32 * (1 + rlse.transpose(1, 2)[..., None].abs())
    tol = (u * (1 + 1e-3) + 2 * es) * pv + u * (1 + 1e-3) * ro.abs()
    if t == torch.float16:
        tol = tol + 2.0 ** -40 * sv + 2.0 ** -25
    worst = float(((o.cpu().double() - ro).abs() / tol).max())
    print(f"  o: {worst:.2f} of its bound", flush=True)
    assert worst <= 1
    assert ((lse.cpu().double() - rlse).abs() <= es.amax(-1).transpose(1, 2)).all()


# ---------------------------------------------------------------- what watches operators, and tensors that are not their memory


def _mock_launches(monkeypatch):
    """The oracle in place of the launches, on CPU tensors, which it takes as the kernels do: by their memory."""
    from dmad_amd import kv_cache

    def tensors(cache, *ts):
        for t in (*ts, *(getattr(cache, n) for n in st.FIELDS)):
            assert t is None or t.numel() == 0 or (t.data_ptr() and not t.is_neg()), "memory that does not hold the values"
        # .data: writes that autograd does not count, as the kernels'
        return {n: None if getattr(cache, n) is None else getattr(cache, n).data for n in st.FIELDS}

    def append(q, k, v, wq, wk, eps, freqs, cache):
        rq, _ = st.append(tensors(cache, q, k, v, wq, wk, freqs), q, k, v, wq, wk, eps, freqs)
        return None if q is None else rq.to(q.dtype)

    def attend(q, cache, scale, causal, accumulate):
        c = tensors(cache, q)
        o, lse, _ = st.attend(c, q, scale=scale, causal=causal, accumulate=accumulate)
        if accumulate:
            cache.weight.data.copy_(c["weight"])
        return o.to(q.dtype), lse.float()

    def evict(cache, keep, recent, sink):
        st.evict(tensors(cache), keep, recent, sink)

    monkeypatch.setattr(kv_cache, "_check_same_device", lambda op, *ts: ts[0].device)
    for name, f in (("_append", append), ("_attend", attend), ("_evict", evict)):
        monkeypatch.setattr(kv_cache, name, f)


BOTH = pytest.mark.parametrize("device", ["cpu", pytest.param("gpu", marks=pytest.mark.gpu)])


def _loop(request, monkeypatch, device, seed=70):
    """A short serving loop's inputs: cache, q, k, v, weights, angles."""
    if device == "cpu":
        _mock_launches(monkeypatch)
    dev = request.getfixturevalue("gpu") if device == "gpu" else torch.device("cpu")
    cache = _make(dev, 2, 2, 16, torch.bfloat16, 16, [37, 20], room=6, seed=seed)
    g = torch.Generator().manual_seed(seed)
    x = dict(q=torch.randn(2, 2, 4, 16, generator=g).bfloat16(), k=torch.randn(2, 2, 2, 16, generator=g).bfloat16(),
             v=torch.randn(2, 2, 2, 16, generator=g).bfloat16(), wq=torch.rand(16, generator=g) + 0.5, wk=torch.rand(16, generator=g) + 0.5,
             freqs=torch.rand(60, 8, generator=g))
    return cache, {n: t.to(dev) for n, t in x.items()}


def _serve(cache, x):
    from dmad_amd import append_kv, evict_low_weight, paged_attention, qk_norm_rope_append

    q = qk_norm_rope_append(x["q"], x["k"], x["v"], x["wq"], x["wk"], 1e-6, x["freqs"], cache)
    o, lse = paged_attention(q, cache, causal=True, accumulate=True, return_lse=True)
    append_kv(x["k"], x["v"], cache)
    evict_low_weight(cache, 24, recent=4, sink=1)
    return [q, o, lse, paged_attention(q, cache)]


@BOTH
@pytest.mark.parametrize("how", ["dispatch mode", "profiled", "compiled", "inference"])
def test_cache_ops_and_direct_calls_agree_bitwise(request, monkeypatch, device, how):
    """The whole loop under what watches operators: the same outputs and the same cache as without."""
    from torch.utils._python_dispatch import TorchDispatchMode

    names = []

    class Names(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            names.append(str(func))
            return func(*args, **(kwargs or {}))

    cache, x = _loop(request, monkeypatch, device)
    want = _serve(cache, x)
    other, x = _loop(request, monkeypatch, device)
    ops = ["qk_norm_rope_append", "paged_attn", "qk_norm_rope_append", "kv_evict", "paged_attn"]
    if how == "dispatch mode":
        with Names():
            got = _serve(other, x)
        assert [n for n in names if "dmad" in n] == [f"dmad.{n}.default" for n in ops]
    elif how == "profiled":
        with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as p:
            got = _serve(other, x)
        assert {f"dmad::{n}" for n in ops} <= {e.key for e in p.key_averages()}
    elif how == "compiled":
        with torch.no_grad():
            got = torch.compile(_serve, fullgraph=True, backend="aot_eager")(other, x)
    else:
        with torch.inference_mode():
            got = _serve(other, x)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    for n in st.FIELDS:
        _same(n, getattr(other, n), getattr(cache, n))


@BOTH
def test_cache_calls_refuse_derivatives(request, monkeypatch, device):
    """Forward-mode tangents and tensors that require a gradient, of the operands and of the cache's own: their
    derivatives would be lost in silence."""
    from dmad_amd import evict_low_weight, paged_attention, qk_norm_rope_append

    cache, x = _loop(request, monkeypatch, device)
    before = st.cache_of(cache)

    def calls(x, cache):
        return [lambda: qk_norm_rope_append(x["q"], x["k"], x["v"], x["wq"], x["wk"], 1e-6, x["freqs"], cache),
                lambda: paged_attention(x["q"], cache), lambda: evict_low_weight(cache, 24)]

    fa = torch.autograd.forward_ad
    with torch.no_grad(), fa.dual_level():
        for name in x:
            for call in calls({**x, name: fa.make_dual(x[name], torch.ones_like(x[name]))}, cache)[:2 if name == "q" else 1]:
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call()
        for name in ("k_pages", "v_pages", "weight"):
            from dmad_amd import PagedKVCache

            t = {n: getattr(cache, n) for n in st.FIELDS}
            dual = PagedKVCache(**{**t, name: fa.make_dual(t[name], torch.ones_like(t[name]))})
            for call in calls(x, dual):
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call()
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda t: paged_attention(t, cache), (x["q"],), (x["q"],))
    for name in ("k_pages", "v_pages", "weight"):
        getattr(cache, name).requires_grad_(True)
        for call in calls(x, cache):
            with pytest.raises(RuntimeError, match="no backward"):
                call()
        getattr(cache, name).requires_grad_(False)
    x["freqs"].requires_grad_(True)
    with pytest.raises(RuntimeError, match="no backward"):
        calls(x, cache)[0]()
    for n in st.FIELDS:
        _same(n, getattr(cache, n), before[n])


@BOTH
def test_cache_calls_read_negated_views(request, monkeypatch, device):
    from dmad_amd import PagedKVCache

    for name in ("q", "k", "v", "wq", "wk", "freqs"):
        cache, x = _loop(request, monkeypatch, device)
        want = _serve(cache, {**x, name: -x[name]})
        other, x = _loop(request, monkeypatch, device)
        for a, b in zip(_serve(other, {**x, name: torch._neg_view(x[name])}), want):
            assert torch.equal(a, b), name
        for n in st.FIELDS:
            _same(n, getattr(other, n), getattr(cache, n))
    # the cache's own tensors are written in place and cannot be such views
    t = {n: getattr(cache, n) for n in st.FIELDS}
    for name in ("k_pages", "weight", "lengths"):
        with pytest.raises(ValueError, match="memory"):
            PagedKVCache(**{**t, name: torch._neg_view(t[name])})
    with pytest.raises(ValueError, match="memory"):
        PagedKVCache(**{**t, "k_pages": torch._efficientzerotensor(t["k_pages"].shape, dtype=torch.bfloat16, device=t["k_pages"].device)})


@BOTH
def test_writes_count_as_changes_in_place(request, monkeypatch, device):
    """A backward pass that saved a view of the pages, lengths or weights before a call that writes them raises; one
    that saved them before a call that only reads them does not."""
    from dmad_amd import append_kv, evict_low_weight, paged_attention

    writes = {"append": {"k_pages", "v_pages", "lengths", "seen", "weight", "position"}, "accumulate": {"weight"},
              "evict": {"k_pages", "v_pages", "lengths", "weight", "position"}, "read": set()}
    for what, names in writes.items():
        cache, x = _loop(request, monkeypatch, device)
        versions = {n: getattr(cache, n)._version for n in st.FIELDS}
        ones = torch.ones((), device=x["q"].device, requires_grad=True)
        kept = {n: (getattr(cache, n)[:1] * ones.to(getattr(cache, n).dtype)).sum() for n in ("k_pages", "v_pages", "weight")}
        if what == "append":
            append_kv(x["k"], x["v"], cache)
        elif what == "evict":
            evict_low_weight(cache, 24)
        else:
            paged_attention(x["q"], cache, accumulate=what == "accumulate")
        for n in st.FIELDS:
            assert (getattr(cache, n)._version != versions[n]) == (n in names), (what, n)
        for n, loss in kept.items():
            if n in names:
                with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                    loss.backward()
            else:
                loss.backward()


@pytest.mark.gpu
def test_caches_made_under_inference_mode(request, monkeypatch):
    """Inference tensors have no count of changes: such a cache works inside and outside the mode."""
    device = "gpu"
    with torch.inference_mode():
        cache, x = _loop(request, monkeypatch, device)
        other, _ = _loop(request, monkeypatch, device)
        assert cache.k_pages.is_inference()
        want = _serve(cache, x)
    with torch.no_grad():
        got = _serve(other, x)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@BOTH
def test_replaced_memory_is_followed(request, monkeypatch, device):
    """A cache tensor whose memory is replaced (.data, as optimizers and offloading do it) is read and written where
    it is now; one without memory, or of another shape or type, is refused by the next call."""
    from dmad_amd import paged_attention

    cache, x = _loop(request, monkeypatch, device)
    other, _ = _loop(request, monkeypatch, device)
    fields = ("k_pages", "v_pages", "page_table", "lengths", "seen", "weight", "position")
    old = {n: getattr(cache, n).data for n in fields}  # kept alive: what a stale address would read and write
    for n in fields:
        getattr(cache, n).data = old[n].clone()
    before = {n: t.clone() for n, t in old.items()}
    for a, b in zip(_serve(cache, x), _serve(other, x)):
        assert torch.equal(a, b)
    for n in fields:
        assert getattr(cache._c, n) == getattr(cache, n).data_ptr() != old[n].data_ptr()
        _same(n, getattr(cache, n), getattr(other, n))
        _same(f"the old {n}", old[n], before[n])
    # a pool of more pages, then what is refused
    for n in ("k_pages", "v_pages", "weight", "position"):
        t = getattr(cache, n)
        t.data = torch.cat((t.data, t.data))
    assert torch.equal(paged_attention(x["q"], cache), paged_attention(x["q"], other)) and cache._c.num_pages == 2 * other._c.num_pages
    good = cache.k_pages.data
    for bad, error in ((good[:3].clone(), ValueError), (good[..., :8].clone(), ValueError), (torch.empty(0, dtype=good.dtype, device=good.device), ValueError)):
        cache.k_pages.data = bad
        with pytest.raises(error):
            paged_attention(x["q"], cache)
    cache.k_pages.data = good
    assert torch.equal(paged_attention(x["q"], cache), paged_attention(x["q"], other))


# ---------------------------------------------------------------- long pieces


def test_oracle_attention_a_head_at_a_time():
    """The oracle for long caches is the one of single tokens and heads."""
    g = torch.Generator().manual_seed(80)
    for causal in (False, True):
        c = dict(k_pages=torch.randn(9, 2, 16, 16, generator=g), v_pages=torch.randn(9, 2, 16, 16, generator=g),
                 page_table=torch.randperm(9, generator=g)[:8].view(2, 4).to(torch.int32), lengths=torch.tensor([2, 60]),
                 seen=torch.tensor([2, 60]), weight=torch.rand(9, 2, 16, generator=g))
        c["page_table"][1, 1] = -1
        d = {n: t.clone() for n, t in c.items()}
        q = torch.randn(2, 3, 4, 16, generator=g)
        a, b = st.attend(c, q, causal=causal, accumulate=True), st.attend_long(d, q, causal=causal, accumulate=True)
        for x, y in zip((*a[:2], *a[2]), (*b[:2], *b[2])):
            assert torch.equal(torch.isinf(x), torch.isinf(y))
            torch.testing.assert_close(x.nan_to_num(0, 0, 0), y.nan_to_num(0, 0, 0), rtol=1e-12, atol=1e-12)
        torch.testing.assert_close(c["weight"], d["weight"], rtol=1e-12, atol=1e-12)


LONG = [
    # S, Hq, Hk, D, dtype, page, lengths, causal, accumulate; tiles of 128 slots per piece, at least
    (1, 40, 40, 128, "bf16", 16, [3000, 1, 700, 5000, 129], False, True, 12),  # pieces over several sequences
    (1, 64, 64, 128, "bf16", 64, [20001], False, False, 33),  # more steps per wave than page ids are looked up at once
    (1, 128, 64, 16, "fp16", 16, [50000], False, True, 33),
    (2, 64, 8, 64, "bf16", 32, [9001, 4000, 30, 12000, 11111, 9090], True, True, 4),
    (4, 64, 8, 64, "fp16", 16, [9001, 4000, 4, 12000, 11111, 9090], True, False, 4),  # two row tiles
    (16, 80, 40, 128, "bf16", 48, [4000, 2500], True, True, 8),  # two row tiles
    (40, 16, 16, 128, "fp16", 16, [5000, 41], True, False, 3),  # two groups of rows
    (3, 32, 32, 256, "bf16", 16, [3000, 2000], True, True, 5),
    (20, 32, 32, 256, "fp16", 64, [2500], True, False, 2),
    (1, 100, 100, 32, "bf16", 128, [9000, 0, 77, 6000], False, False, 20),
    (1, 64, 64, 16, "bf16", 16, [(97 * i) % 900 for i in range(130)], False, True, 30),  # more than 64 sequences
]


def _tiles_per_piece(Hk, D, page, S, Hq, lengths, room):
    """Tiles that a piece of the attention covers: the number of pieces from the scratch that it asks for."""
    from dmad_amd import _native as nat

    B, M = len(lengths), -(-(max(lengths) + room) // page)
    c = _c_cache(nat, num_pages=B * M, kv_heads=Hk, page_size=page, head_dim=D, batch=B, pages_per_seq=M, table_stride=M,
                 ks=(Hk * page * D, page * D, D), vs=(Hk * page * D, page * D, D))
    row = Hk * (S * Hq // Hk) * (4 * D + 8)
    pieces = (nat.paged_attn_workspace_bytes(c, S, Hq, False) - 512) // row - B  # the two parts are rounded up to 256
    tiles = sum(max(1, -(-n // 128)) for n in lengths)
    return -(-tiles // (pieces + 1)), pieces


@pytest.mark.parametrize("S,Hq,Hk,D,dtype,page,lengths,causal,accumulate,least", LONG)
def test_long_cases_have_long_pieces(S, Hq, Hk, D, dtype, page, lengths, causal, accumulate, least):
    """A wave takes one step of 32 slots per tile: these cases run the attention's loop, not its last step alone."""
    per_piece, pieces = _tiles_per_piece(Hk, D, page, S, Hq, lengths, 5)
    assert per_piece >= least, (per_piece, pieces)


@pytest.mark.gpu
@pytest.mark.parametrize("S,Hq,Hk,D,dtype,page,lengths,causal,accumulate,least", LONG)
def test_attention_of_long_pieces(gpu, S, Hq, Hk, D, dtype, page, lengths, causal, accumulate, least):
    from dmad_amd import paged_attention

    B, t = len(lengths), DTYPES[dtype]
    print(f"case long B={B} S={S} Hq={Hq} Hk={Hk} D={D} {dtype} page={page} lengths={lengths[:4]} causal={causal}", flush=True)
    cache = _make(gpu, B, Hk, D, t, page, lengths, room=5, seed=D + S)
    # whole pages missing inside pieces, one of them in the last, and an id beyond the pool
    longest = lengths.index(max(lengths))
    cache.page_table[longest, [3, 17, (max(lengths) - 1) // page // 2]] = torch.tensor([-1, cache.k_pages.shape[0], -7], dtype=torch.int32, device=gpu)
    q = (torch.randn(B, S, Hq, D, generator=torch.Generator().manual_seed(1)) * 1.5).to(t).to(gpu)
    c = {n: getattr(cache, n) for n in st.FIELDS}
    before = cache.weight.clone()
    ref = st.attend_long(c, q, causal=causal, accumulate=accumulate)
    got = paged_attention(q, cache, causal=causal, accumulate=accumulate, return_lse=True)
    torch.cuda.synchronize()
    ro, rlse, bound = ref[0].cpu(), ref[1].cpu(), tuple(x.cpu() for x in ref[2])
    _check_attention(got, (ro, rlse, bound), t, D)
    if accumulate:
        w, r = cache.weight.cpu().double(), c["weight"].cpu()
        _same("weights of unused slots", torch.isnan(w).float(), torch.isnan(r).float())
        share = (r - before.cpu().double()).nan_to_num(0)
        worst = float(bound[2].max()) * (D + 8) * F32 * 2 + 128 * F32 * (1 + float(rlse[~torch.isinf(rlse)].abs().max()))
        assert ((w - r).abs().nan_to_num(0) <= worst * share + 2 * F32 * r.abs().nan_to_num(0) + 1e-30).all()
    for _ in range(2):
        assert torch.equal(paged_attention(q, cache, causal=causal), got[0])


@pytest.mark.gpu
@pytest.mark.parametrize("S,Hq,Hk,D,dtype,lengths", [(4, 64, 64, 128, "bf16", [3000, 2000]), (3, 128, 64, 64, "fp16", [4000]),
                                                     (5, 40, 40, 256, "bf16", [2600]), (17, 80, 40, 32, "fp16", [70, 5000])])
def test_hidden_tokens_after_long_pieces(gpu, S, Hq, Hk, D, dtype, lengths):
    """Infinities and NaN in the new tokens' values, behind many steps that need no mask: they reach the tokens that
    see them, of their key head and sequence, and no other."""
    from dmad_amd import paged_attention

    B, t, G = len(lengths), DTYPES[dtype], Hq // Hk
    assert _tiles_per_piece(Hk, D, 16, S, Hq, lengths, 0)[0] >= 3
    cache = _make(gpu, B, Hk, D, t, 16, lengths, seed=90 + D)
    q = torch.randn(B, S, Hq, D, generator=torch.Generator().manual_seed(3)).to(t).to(gpu)
    clean = paged_attention(q, cache, causal=True)
    ref = st.attend_long({n: getattr(cache, n) for n in st.FIELDS}, q, causal=True)
    _check_attention((clean, ref[1].float()), (ref[0].cpu(), ref[1].cpu(), tuple(x.cpu() for x in ref[2])), t, D)
    head = Hk // 2
    rows = slice(head * G, head * G + G)
    for token in (0, 1, S - 1):
        for name, value in (("v_pages", math.inf), ("v_pages", math.nan), ("k_pages", math.nan)):
            page, slot = st.locate(st.cache_of(cache), B - 1, lengths[-1] - S + token)
            pages = getattr(cache, name)
            keep = pages[page, head, slot].clone()
            pages[page, head, slot] = value
            o = paged_attention(q, cache, causal=True)
            assert not torch.isfinite(o[-1, token:, rows].float()).any(), (token, name)
            o[-1, token:, rows] = clean[-1, token:, rows]
            assert torch.equal(o, clean), (token, name)
            pages[page, head, slot] = keep


@pytest.mark.gpu
@pytest.mark.parametrize("B,Hk,D,page,length,keep", [(4, 32, 256, 16, 900, 420), (130, 40, 128, 16, 44, 20), (1, 5, 64, 48, 7000, 33)])
def test_evict_more_rows_than_workgroups(gpu, B, Hk, D, page, length, keep):
    """Copies whose workgroups take several rows each, and a capacity of which nearly nothing moves."""
    from dmad_amd import evict_low_weight

    cache = _make(gpu, B, Hk, D, torch.bfloat16, page, [length - b % 7 for b in range(B)], seed=keep)
    c = st.cache_of(cache)
    st.evict(c, keep, 5, 1)
    evict_low_weight(cache, keep, recent=5, sink=1)
    torch.cuda.synchronize()
    for n in st.FIELDS:
        _same(n, getattr(cache, n), c[n])
    cache.lengths.fill_(keep)  # nothing to cut
    c = st.cache_of(cache)
    evict_low_weight(cache, keep, recent=5)
    for n in st.FIELDS:
        _same(n, getattr(cache, n), c[n])


# ---------------------------------------------------------------- a student of this package, block by block


def test_the_tangent_module_names_the_cache():
    from types import SimpleNamespace

    from dmad_amd import MinimalA2AAttnOpWithT

    with pytest.raises(NotImplementedError, match="PagedKVCache"):
        MinimalA2AAttnOpWithT()(None, None, None, attn_ctx=SimpleNamespace(rope=None, kv_cache=object(), mode="APPEND"))


@pytest.mark.gpu
def test_a_student_that_norms_over_the_width(gpu):
    """Queries and keys normalised over the model width and rotated by the prologue, block after block into the
    cache: each block attends to itself and what came before, as the dense attention does over the same keys."""
    from dmad_amd import PagedKVCache, append_kv, paged_attention, plain_attention, rmsnorm_rope_with_tangent

    B, block, blocks, H, D = 2, 24, 4, 4, 64
    g = torch.Generator().manual_seed(40)
    qkv = torch.randn(B, block * blocks, 3, H * D, generator=g).bfloat16().to(gpu)
    wq, wk = ((1 + 0.2 * torch.randn(H * D, generator=g)).bfloat16().to(gpu) for _ in range(2))
    freqs = (torch.rand(block * blocks, D // 2, generator=g) * 50).to(gpu)
    cache = PagedKVCache.allocate(B, block * blocks, H, D, device=gpu, page_size=16, track_weights=False)
    keys, values = [], []
    for i in range(blocks):
        at = slice(i * block, (i + 1) * block)
        y = qkv[:, at].contiguous()
        with torch.no_grad():
            q, _ = rmsnorm_rope_with_tangent((y[:, :, 0].contiguous(), None), wq, 1e-6, freqs[at], H)
            k, _ = rmsnorm_rope_with_tangent((y[:, :, 1].contiguous(), None), wk, 1e-6, freqs[at], H)
        v = y[:, :, 2].reshape(B, block, H, D)
        append_kv(k, v, cache)
        ref = st.attend(st.cache_of(cache), q.cpu())
        got = paged_attention(q, cache, return_lse=True)
        _check_attention(got, ref, torch.bfloat16, D)
        keys.append(k), values.append(v)
        dense = plain_attention(*(x.transpose(1, 2).contiguous() for x in (q, torch.cat(keys, 1), torch.cat(values, 1))))
        dense = dense.transpose(1, 2).float()
        assert float((got[0].float() - dense).norm() / dense.norm()) < 5e-3
    assert cache.lengths.tolist() == cache.seen.tolist() == [block * blocks] * B


@BOTH
def test_one_memory_for_two_tensors_is_not_written(request, monkeypatch, device):
    """lengths given as seen too ("equal until something is evicted") would advance twice per token, and keys and
    values in one memory overwrite each other: refused by what writes, fine for what reads."""
    from dmad_amd import PagedKVCache, append_kv, evict_low_weight, paged_attention

    cache, x = _loop(request, monkeypatch, device)
    t = {n: getattr(cache, n) for n in st.FIELDS}
    both = torch.zeros(3, device=t["lengths"].device, dtype=torch.int32)
    both[:2] = t["lengths"]
    want = paged_attention(x["q"], cache)
    for over, match in ((dict(seen=t["lengths"]), "lengths and seen"), (dict(lengths=both[:2], seen=both[1:]), "lengths and seen"),
                        (dict(v_pages=t["k_pages"]), "k_pages and v_pages")):
        same = PagedKVCache(**{**t, **over})
        before = st.cache_of(same)
        with pytest.raises(ValueError, match=match):
            append_kv(x["k"], x["v"], same)
        with pytest.raises(ValueError, match=match):
            evict_low_weight(same, 24)
        if "v_pages" not in over:
            assert torch.equal(paged_attention(x["q"], same), want)
        for n in st.FIELDS:
            _same(n, getattr(same, n), before[n])
    counts = torch.stack([t["lengths"], t["seen"]])  # beside each other in one tensor
    append_kv(x["k"], x["v"], PagedKVCache(**{**t, "lengths": counts[0], "seen": counts[1]}))
    assert counts[0].tolist() == [39, 22] and counts[1].tolist() == [39, 22]


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["qk_norm_rope_append", "append without q", "paged_attn", "paged_attn weights", "kv_evict"])
def test_registered_ops_do_what_they_declare(gpu, op):
    """torch's own checks: what is written is what the schema names, and the shapes are those of the fakes."""
    from dmad_amd import PagedKVCache

    cache = PagedKVCache.allocate(2, 64, 2, 16, device=gpu, page_size=16)
    g = torch.Generator().manual_seed(95)
    for n in ("k_pages", "v_pages"):
        getattr(cache, n).copy_(torch.randn(cache.k_pages.shape, generator=g))
    cache.weight.copy_(torch.rand(cache.weight.shape, generator=g))
    cache.position.copy_(torch.arange(cache.position.numel()).view_as(cache.position) % 50)
    cache.lengths.fill_(40), cache.seen.fill_(40)
    c = [getattr(cache, n) for n in ("k_pages", "v_pages", "page_table", "lengths", "seen", "weight", "position")]
    q, k = (torch.randn(2, 3, h, 16, generator=g).bfloat16().to(gpu) for h in (4, 2))
    w, f = torch.ones(16, device=gpu), torch.rand(60, 8, generator=g).to(gpu)
    args = {"qk_norm_rope_append": (q, k, k.clone(), w, None, 1e-6, f, *c), "append without q": (None, k, k.clone(), None, None, 0.0, None, *c),
            "paged_attn": (q, 0.25, True, *c[:5], None, None), "paged_attn weights": (q, 0.25, False, *c), "kv_evict": (20, 3, 1, *c)}[op]
    name = {"append without q": "qk_norm_rope_append", "paged_attn weights": "paged_attn"}.get(op, op)
    torch.library.opcheck(getattr(torch.ops.dmad, name).default, args, test_utils=("test_schema", "test_faketensor", "test_aot_dispatch_dynamic"))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_subnormal_keys_and_values(gpu, dtype):
    """Keys and values below the type's smallest normal are not flushed."""
    from dmad_amd import paged_attention

    t = DTYPES[dtype]
    for which in ("k_pages", "v_pages"):
        cache = _make(gpu, 1, 1, 32, t, 16, [90], seed=96)
        tiny = torch.finfo(t).smallest_normal
        getattr(cache, which).copy_((torch.rand(cache.k_pages.shape, generator=torch.Generator().manual_seed(97)) * tiny).to(t))
        q = torch.randn(1, 1, 2, 32, generator=torch.Generator().manual_seed(98)).to(t)
        scale = 0.2 if which == "v_pages" else min(0.2 / tiny, 2.0 ** 126)
        ref = st.attend(st.cache_of(cache), q, scale=scale)
        o, lse = paged_attention(q.to(gpu), cache, sm_scale=scale, return_lse=True)
        u, step = torch.finfo(t).eps / 2, tiny * torch.finfo(t).eps / 2
        es = (32 + 8) * F32 * ref[2][2] + 64 * F32 * (1 + ref[1].transpose(1, 2)[..., None].abs())
        tol = (u + 2 * es) * 1.001 * ref[2][0] + u * ref[0].abs() + step
        if t == torch.float16:
            tol = tol + 2.0 ** -40 * ref[2][1]
        assert ((o.cpu().double() - ref[0]).abs() <= tol).all() and float(ref[0].abs().max()) > 0
        assert ((lse.cpu().double() - ref[1]).abs() <= es.amax(-1).transpose(1, 2)).all()


@BOTH
def test_registered_ops_refuse_what_the_calls_refuse(request, monkeypatch, device):
    """The registered ops check what they are given as the calls do, before a kernel reads it."""
    cache, x = _loop(request, monkeypatch, device)
    c = [getattr(cache, n) for n in ("k_pages", "v_pages", "page_table", "lengths", "seen", "weight", "position")]
    before = st.cache_of(cache)
    append, attend, evict = (getattr(torch.ops.dmad, n) for n in ("qk_norm_rope_append", "paged_attn", "kv_evict"))
    q, k, v, wq, wk, f = (x[n] for n in ("q", "k", "v", "wq", "wk", "freqs"))
    for call in [
        lambda: append(q[:1], k, v, wq, wk, 1e-6, f, *c), lambda: append(q, k, v[:, :1], wq, wk, 1e-6, f, *c),
        lambda: append(q, k[:, :, :1], v, wq, wk, 1e-6, f, *c), lambda: append(q, k.half(), v, wq, wk, 1e-6, f, *c),
        lambda: append(q, k, v, wq, wk, 1e-6, f[:, :4], *c), lambda: append(q, k, v, wq, wk, -1.0, f, *c),
        lambda: append(q, k, v, wq, wk, 1e-6, f, *c[:3], c[3][:1], *c[4:]),
        lambda: attend(q[..., :8], 0.25, False, *c), lambda: attend(q[:, :, :3], 0.25, False, *c),
        lambda: attend(q, 0.25, False, c[0][:2], *c[1:]), lambda: attend(q[:1], 0.25, True, *c[:5], None, None),
        lambda: evict(0, 0, 0, *c), lambda: evict(8, 5, 4, *c), lambda: evict(8, 0, 0, *c[:5], c[5][:1], c[6]),
    ]:
        with pytest.raises(ValueError):
            call()
    with pytest.raises(NotImplementedError):
        attend(q, -0.25, False, *c)
    for n in st.FIELDS:
        _same(n, getattr(cache, n), before[n])
