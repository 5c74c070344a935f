"""The serving library without a GPU: its header, its refusals, and the index arithmetic of its kernels."""
import ctypes as C
import re
import shutil
import subprocess
import struct
from pathlib import Path

import pytest
import torch

import serving_cases as S

ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def lib():
    from dejavu_b200 import _lib, build

    build.build()
    return _lib.load_serving()


def test_library_matches_its_header(lib):
    from dejavu_b200 import _lib

    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "dejavu_b200_serving.h").read_text(), flags=re.S)
    names = sorted(set(re.findall(r"\b(djv_[a-z0-9_]+)\s*\(", text)))
    assert sorted(_lib.SERVING_SIGNATURES) == names and "djv_sample" in names
    for name in names:
        assert hasattr(lib, name)
        declared = re.search(rf"\b{name}\s*\((.*?)\)", text, flags=re.S).group(1)
        args = [] if declared.strip() == "void" else declared.split(",")
        kinds = [C.c_void_p if "*" in a else {"int": C.c_int, "long long": C.c_longlong, "float": C.c_float, "size_t": C.c_size_t}
                 [re.sub(r"\s+\w+$", "", a.strip())] if " " in a.strip() else C.c_int for a in args]
        assert _lib.SERVING_SIGNATURES[name][1] == kinds, name
    assert lib.djv_version() >= 100


def bits(x):
    return struct.unpack("q", struct.pack("d", x))[0]


P = 1 << 20  # an aligned address that nobody reads


def append(lib, dtype=1, q_out=P, k=P, pages_at=P, ld_page=4096, pages=4, page=16, width=3, freqs=P, half=32, B=2, T=2, H=4, G=2, D=64, cu=None):
    return lib.djv_paged_append(dtype, q_out, None, P, 256, 64, k, 128, 64, P, 128, 64, pages_at, P, ld_page, 1024, 64, pages, page, P, 3, width,
                                P, cu, freqs, 1.0, half, 0, B, T, H, G, D, None)


def attend(lib, dtype=1, q=P, ldq=256, pages_at=P, page=16, width=3, B=2, H=4, G=2, D=64, scale=0.1, scratch=P, size=1 << 30):
    return lib.djv_paged_attention(dtype, P, q, ldq, 64, pages_at, P, 4096, 1024, 64, 4, page, P, 3, width, P, B, H, G, D, scale, scratch, size,
                                   None)


def packed(lib, dtype=1, out=P, cu=P, B=2, T=9, H=4, G=2, D=64, scale=0.1):
    return lib.djv_packed_attention(dtype, out, P, 256, 64, P, 128, 64, P, 128, 64, cu, B, T, H, G, D, scale, 0, None)


def sample(lib, dtype=2, logits=P, ld=100, t=1.0, k=0, p=1.0, m=0.0, B=2, V=100):
    return lib.djv_sample(dtype, P, logits, ld, P, None, bits(t), None, k, None, bits(p), None, bits(m), B, V, None)


@pytest.mark.parametrize("call,arguments", [(f, a) for f, many in {
    append: [{"dtype": 3}, {"k": None}, {"pages_at": P + 8}, {"ld_page": 4100}, {"pages": 0}, {"page": 0}, {"width": 0}, {"freqs": None},
             {"half": 33}, {"half": -1}, {"B": 0}, {"T": 3}, {"T": -1}, {"H": 0}, {"G": 0}, {"D": 60}, {"D": 0}, {"D": 4096},
             {"page": 1 << 20, "width": 1 << 12}],
    attend: [{"dtype": -1}, {"q": None}, {"q": P + 4}, {"ldq": 257}, {"pages_at": P + 2}, {"H": 5}, {"H": 0}, {"D": 264}, {"D": 12}, {"B": -1},
             {"scale": float("nan")}, {"scale": float("inf")}, {"page": 1 << 20, "width": 1 << 12}],
    packed: [{"dtype": 7}, {"out": None}, {"cu": None}, {"B": 0}, {"T": -1}, {"H": 3}, {"G": 0}, {"D": 0}, {"D": 257}, {"scale": float("inf")},
             {"scale": float("nan")}],
    sample: [{"dtype": 9}, {"logits": None}, {"ld": 99}, {"t": -0.5}, {"t": float("nan")}, {"t": float("inf")}, {"k": -1}, {"p": -0.1},
             {"p": float("nan")}, {"m": 1.5}, {"m": -1.0}, {"m": float("nan")}, {"V": 0}, {"B": -1}]}.items() for a in many], ids=str)
def test_kernels_check_their_arguments_on_the_host(lib, call, arguments):
    """Nothing is launched: there is no GPU."""
    from dejavu_b200 import _lib

    before = lib.djv_launch_count()
    assert call(lib, **arguments) == _lib.ERR_INVALID and lib.djv_last_error() and lib.djv_launch_count() == before


def test_nothing_to_do_is_no_launch(lib):
    before = lib.djv_launch_count()
    assert append(lib, T=0, cu=P) == attend(lib, B=0) == packed(lib, T=0) == sample(lib, B=0) == 0 and lib.djv_launch_count() == before


def test_operators_refuse_tensors_of_the_cpu():
    from dejavu_b200 import ops

    bf16 = torch.bfloat16
    q, k, pages = torch.zeros(2, 4, 64, dtype=bf16), torch.zeros(2, 2, 64, dtype=bf16), torch.zeros(3, 2, 16, 64, dtype=bf16)
    table, pos, cu = torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int64), torch.tensor([0, 1, 2], dtype=torch.int32)
    for call in (lambda: ops.paged_append(q, k, k, pages, pages, table, pos), lambda: ops.paged_attention(q, pages, pages, table, pos, 0.1),
                 lambda: ops.packed_attention(q, k, k, cu, 0.1), lambda: ops.sample_tokens(q[:, 0], torch.zeros(2))):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()


def compiled(tmp_path, body):
    (tmp_path / "t.cpp").write_text(f'#include "{ROOT}/dejavu_b200/csrc/serving_plan.cuh"\n#include <stdio.h>\n#include <limits.h>\n#include <initializer_list>\n'
                                    "#define CHECK(c) if (!(c)) { printf(\"%s line %d\\n\", #c, __LINE__); return 1; }\nusing namespace djv;\n"
                                    "int main() {\n" + body + "\nreturn 0;\n}\n")
    subprocess.run([shutil.which("g++"), "-std=c++17", "-O1", "-fsanitize=address,undefined", str(tmp_path / "t.cpp"), "-o", str(tmp_path / "t")],
                   check=True)
    r = subprocess.run([str(tmp_path / "t")], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr


def test_pages_of_tokens(tmp_path):
    """A page is inside the pool or none, whatever the table holds and whatever position is asked for."""
    compiled(tmp_path, """
  const int table[6] = {3, -1, 9, 10, INT_MAX, INT_MIN};
  for (int page : {1, 3, 16, 1000}) {
    const PageMap m{table, 6, page, 10, divider_of(page)};
    const long long want[6] = {3, NO_PAGE, 9, NO_PAGE, NO_PAGE, NO_PAGE};
    for (long long t = 0; t < 6ll * page; ++t) {
      int slot;
      CHECK(page_of(m, t, slot) == want[t / page] && slot == t % page)
    }
    for (long long t : {6ll * page, 6ll * page + 1, 1ll << 33, LLONG_MAX, -1ll, LLONG_MIN}) {
      int slot;
      CHECK(page_of(m, t, slot) == NO_PAGE)
    }
  }""")


def test_division_by_a_page(tmp_path):
    compiled(tmp_path, """
  unsigned r = 12345;
  for (unsigned d = 1; d < 5000; ++d) {
    const Divider v = divider_of(d);
    for (unsigned t = 0; t < 300; ++t) CHECK(divided(t, v) == t / d)
    for (unsigned k = 1; k < 40; ++k)
      for (int e = -1; e <= 1; ++e) {
        const unsigned t = (unsigned)(((unsigned long long)d * k * 997 + e) % 0x7fffffffu);
        CHECK(divided(t, v) == t / d)
      }
    for (unsigned t : {0x7fffffffu, 0x7ffffffeu, 0x7fffffffu / d * d, 0x7fffffffu / d * d - 1}) CHECK(divided(t, v) == t / d)
  }
  for (int i = 0; i < 2000000; ++i) {
    r = r * 1664525u + 1013904223u;
    const unsigned d = (r >> (r % 31)) % 0x7fffffffu + 1;
    r = r * 1664525u + 1013904223u;
    const unsigned t = r >> 1;
    CHECK(divided(t, divider_of(d)) == t / d)
  }""")


def test_sequences_of_rows(tmp_path):
    """The last sequence that does not begin after a row, found as a warp does; with offsets that make no sense still one of the batch,
    and no offset is looked at but theirs."""
    compiled(tmp_path, """
  auto find = [](const int *cu, int B, int t) {
    SequenceSearch s{0, B};
    for (int n = 0; !s.done(); ++n) {
      if (n > 40) return -2;
      int before = 0;
      for (int lane = 0; lane < 32; ++lane)
        if (s.probe(lane) < s.hi && cu[s.probe(lane)] <= t) before = lane + 1;
      s.narrow(before);
    }
    return s.lo;
  };
  const int cu[7] = {2, 2, 5, 5, 5, 11, 12};
  for (int t = 2; t < 12; ++t) {
    int want = -1;
    for (int b = 0; b < 6; ++b)
      if (cu[b] <= t && t < cu[b + 1]) want = b;
    CHECK(find(cu, 6, t) == want)
  }
  static int many[100001];
  for (int B : {1, 31, 32, 33, 1000, 1025, 100000}) {
    for (int b = 0; b <= B; ++b) many[b] = b / 3 * 7;
    for (int t = 0; t < many[B]; t += 1 + B / 500) {
      const int b = find(many, B, t);
      CHECK(b >= 0 && b < B && many[b] <= t && t < many[b + 1])
    }
  }
  const int odd[4][4] = {{0, 9, 3, 20}, {5, -7, 30, 6}, {INT_MIN, 8, INT_MIN, INT_MAX}, {9, 9, 9, 9}};
  for (auto &o : odd)
    for (int t = 0; t < 20; ++t) {
      const int b = find(o, 3, t);
      CHECK(b >= 0 && b < 3)
    }""")


def test_definitions_agree_with_torch():
    g = torch.Generator().manual_seed(1)
    row = torch.randn(50, generator=g, dtype=torch.float64)
    n, p = 20000, torch.softmax(row / 0.7, 0)
    got = torch.tensor([S.sample(row, (i + 0.5) / n, 0.7, 0, 1.0, 0.0) for i in range(0, n, 10)]).bincount(minlength=50) * 10 / n
    assert float((got - p).abs().max()) <= 2 * 10 / n
    first = row.argsort(descending=True)
    assert {S.sample(row, i / 100, 0.7, 3, 1.0, 0.0) for i in range(100)} <= set(first[:3].tolist())
    assert S.sample(row, 0.99, 0.7, 0, 0.0, 0.0) == S.sample(row, 0.5, 0.0, 0, 1.0, 0.0) == first[0]
    q, k, v = (torch.randn(n, 8, generator=g, dtype=torch.float64) for n in (3, 5, 5))
    want = torch.nn.functional.scaled_dot_product_attention(q[None], k[None], v[None], scale=0.3)[0]
    assert torch.allclose(S.attend(q, k, v, 0.3)[0], want, rtol=1e-12)
    x, f = torch.randn(2, 6, generator=g, dtype=torch.float64), torch.tensor([0.5, 0.25])
    y, _ = S.rotate(x, 7, f, 2.0, True)
    turn = torch.polar(torch.full((2,), 2.0, dtype=torch.float64), 7 * f.double())
    want = torch.view_as_real(torch.view_as_complex(x[:, :4].reshape(2, 2, 2)) * turn).flatten(1)
    assert torch.allclose(y[:, :4], want) and torch.equal(y[:, 4:], x[:, 4:])


def test_units_of_a_batch_are_dealt_out_once(tmp_path):
    """Every unit of every item belongs to one block, in order; parts stay inside their item; an item that is split has one beginning and
    one end, and the block after a part's block goes on where it stopped."""
    compiled(tmp_path, """
  const long long lengths[5][4] = {{1, 1, 1, 1}, {0, 64, 65, 5000}, {100000, 1, 0, 7}, {640, 640, 640, 640}, {0, 0, 0, 0}};
  for (auto &tokens : lengths)
    for (int share : {1, 3, 8})
      for (int blocks : {1, 2, 7, 296})
        for (int least : {1, 4}) {
          long long total = 0, base[4];
          for (int b = 0; b < 4; ++b) {
            base[b] = total;
            const long long u = units_of(tokens[b]);
            CHECK(u >= 1 && tokens_before(0, tokens[b]) == 0 && tokens_before(DECODE_ITEM, tokens[b]) == 0 && tokens_before(u, tokens[b]) == tokens[b])
            for (long long i = 0; i < u; ++i) {
              const long long n = tokens_before(i + 1, tokens[b]) - tokens_before(i, tokens[b]);
              CHECK(n >= (i >= DECODE_ITEM) && n <= (i >= DECODE_ITEM ? DECODE_UNIT : 0))
            }
            total += units_of(tokens[b]) * share;
          }
          const long long per = units_per_block(total, blocks, least);
          CHECK(per >= least && per * blocks >= total)
          long long at = 0;
          for (int c = 0; c < blocks; ++c) {
            long long x = c * per;
            const long long end = x + per < total ? x + per : total;
            if (x >= end) continue;
            int b = 3;
            while (base[b] > x) --b;
            while (x < end) {
              const long long units = units_of(tokens[b]);
              const DecodePart p = decode_part(x, end, base[b], units);
              CHECK(x == at && p.item >= 0 && p.item < share && p.from >= 0 && p.from < p.to && p.to <= units)
              CHECK(base[b] + p.item * units + p.from == x)
              x += p.to - p.from;
              at = x;
              CHECK(p.to == units || x == end)
              if (x < end && x == base[b] + units * share) ++b;
            }
          }
          CHECK(at == total)
        }""")
