"""CPU test of how the attention over shared prefixes cuts what a plan says to what
there is (hy-mt-rs_amd/csrc/hyq_paged_pieces.hpp, compiled here with g++): plans of
any bytes, whose every row, place, page entry and part must lie inside its buffer
and whose every loop must end."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "hy-mt-rs_amd", "csrc", "hyq_paged_pieces.hpp")

PROGRAM = r'''
#include "HEADER"
#include <climits>
#include <cstdio>
#include <random>
using namespace hyq;
static int fails = 0;
#define CHECK(c) do { if (!(c) && fails++ < 20) std::printf("line %d: %s\n", __LINE__, #c); } while (0)
static std::mt19937 rng(1);
static int below(int n) { return (int)(rng() % (unsigned)n); }
// a number of a plan: any bits, an end of the range, or a small one
static int any(int most)
{
    switch (below(5)) {
    case 0: return (int)rng();
    case 1: return below(2) ? INT_MAX - below(3) : INT_MIN + below(3);
    case 2: return below(2 * most + 2) - 2;
    case 3: return -1 - below(40);
    default: return below(64);
    }
}
// the page entries of the steps from position p on, 16 positions each
static void entries(const PlanSizes &z, int p, int len)
{
    const long long at = (long long)p >> z.shift;
    CHECK(p >= 0 && (p & 15) == 0);
    if (p < len) CHECK(at < z.stride);
    CHECK((p & ((1 << z.shift) - 1)) + 15 < 1 << z.shift);
}
int main()
{
    for (int i = 0; i < 400000; ++i) {
        const int rep = 1 + below(16), few = 16 / rep;
        PlanSizes z{};
        z.seqs = 1 + below(below(2) ? 5 : 4096), z.kvh = 1 + below(below(2) ? 4 : 256);
        z.rows = 1 + below(below(2) ? 9 : 1 << 20), z.shift = 4 + below(5);
        z.stride = 1 + below(below(2) ? 6 : 1 << (24 - z.shift));
        z.tq = 128 / rep, z.cap = z.seqs / 8 + z.seqs / 2 + 1;
        z.most = z.cap + 256 / z.kvh + 1;
        z.few_most = (2048 + (z.seqs + z.cap) * z.kvh + 1023) / 1024 * 1024;
        const int big = below(2) ? z.few_most : z.rows;
        const int tile = below(2) ? 16 : 32;

        FewPiece f{any(z.seqs), any(z.kvh), any(100), any(100), any(big), any(20), any(5000),
                   any(5000), any(9), any(2), {}};
        f = cut_few_piece(z, tile, f);
        CHECK(f.slot >= 0 && f.slot < z.seqs && f.kh >= 0 && f.kh < z.kvh);
        const int places = f.narrow ? z.cap * z.tq : z.rows;
        CHECK(f.n >= 0 && f.begin >= 0 && f.begin < places && f.begin + f.n <= places);
        // (a slot of more rows than the form takes is left out)
        if (f.narrow) CHECK(f.n <= few);
        if (f.n <= few)
            for (int c = 0; c < 16; ++c) {
                const bool ok = c / rep < f.n;
                CHECK(f.begin + (ok ? c / rep : 0) < places);
                if (ok) CHECK(c < few * rep); // (a row of its part)
            }
        CHECK(f.len >= 0 && f.len <= z.positions() && f.skip >= 0 && f.skip <= f.len);
        CHECK(f.t0 >= 0 && f.t1 > f.t0);
        CHECK((long long)f.skip + (long long)f.t1 * tile < (long long)f.len + 2 * tile);
        for (int t : {f.t0, f.t1 - 1})
            for (int p = f.skip + t * tile; p < f.skip + (t + 1) * tile; p += 16)
                entries(z, p, f.len);

        Piece p{any(z.seqs), any(z.cap), any(100), any(100), any(z.most), any(9), any(200), any(5000)};
        p = cut_piece(z, 64, p);
        CHECK(p.slot >= 0 && p.slot < z.seqs && p.part >= 0 && p.part < z.most);
        CHECK(p.index >= 0 && p.index < z.cap); // (its list: index * tq .. + tq - 1)
        CHECK(p.first >= 0 && p.first <= z.positions());
        CHECK(p.t0 >= 0 && p.t0 * 64 <= p.first && p.t1 >= 0 && p.t1 * 64 <= p.first + 64);
        for (int at = p.t0 * 64; at < p.t0 * 64 + 64; at += 16)
            entries(z, at, p.first);

        for (bool narrow : {false, true}) {
            const SharedPlace any_place{any(big), any(20), any(big), any(90), any(130), any(big),
                                        any(90), 0};
            for (int kh : {0, z.kvh - 1}) {
                const SharedPlace s = cut_place(z, kh, narrow, any_place);
                CHECK(s.begin >= 0 && s.n >= 0 && s.begin + s.n <= z.rows);
                CHECK(s.first >= 0 && s.ways >= 0 && s.first + s.ways <= z.few_most);
                CHECK(s.part >= 0 && s.pieces >= 0);
                CHECK(s.part + s.pieces <= (narrow ? z.few_most : z.most));
            }
        }
        // what a plan of the batch says stays as it is
        const int len = (int)(z.positions() < 64 ? z.positions() : 64 + below((int)z.positions() - 63));
        const int skip = (len - 1) >> z.shift << z.shift, tiles = (len - skip + tile - 1) / tile;
        const FewPiece own{below(z.seqs), below(z.kvh), 0, tiles, below(z.rows), 1, len, skip, 1, 0, {}};
        const FewPiece kept = cut_few_piece(z, tile, own);
        CHECK(kept.slot == own.slot && kept.kh == own.kh && kept.t0 == 0 && kept.t1 == tiles);
        CHECK(kept.begin == own.begin && kept.n == 1 && kept.len == len && kept.skip == skip);
    }
    std::printf("%d\n", fails);
    return fails != 0;
}
'''


def test_plans_of_any_bytes_stay_inside(tmp_path):
    src, exe = tmp_path / "pieces.cpp", tmp_path / "pieces"
    src.write_text(PROGRAM.replace("HEADER", HEADER))
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout + out.stderr
