"""The division of chunk attention's work among workers, run on the CPU: the kernels' own device functions compiled for the
host, a warp as 32 threads.  Every key tile of every item belongs to one worker; and where lengths change under a
kernel (a caller's mistake) a worker's run ends inside the tables, whatever it reads."""
import os
import random
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "inference-project_b200", "csrc")

# what k_attn_chunk.cuh takes from common.cuh and the CUDA headers
STUB = r"""
#pragma once
#include <math.h>
#include <stdint.h>
#include <string.h>
#include <algorithm>
#include <barrier>
#define __device__
#define __global__
#define __host__
#define __shared__
#define __forceinline__ inline
#define __align__(n) __attribute__((aligned(n)))
#define __launch_bounds__(...)
struct Dim { unsigned x, y; };
inline thread_local Dim threadIdx;
inline Dim blockIdx, blockDim = {32, 1};
inline std::barrier<> bar(32);
inline uint64_t lane_word[32];
inline void __syncthreads() { bar.arrive_and_wait(); }
inline void __syncwarp() { bar.arrive_and_wait(); }
template <typename T> T from_lane(T v, int lane)
{
	memcpy(&lane_word[threadIdx.x], &v, sizeof v);
	bar.arrive_and_wait();
	T r;
	memcpy(&r, &lane_word[lane], sizeof r);
	bar.arrive_and_wait();
	return r;
}
template <typename T> T __shfl_sync(unsigned, T v, int lane) { return from_lane(v, lane); }
template <typename T> T __shfl_up_sync(unsigned, T v, int o) { return from_lane(v, (int)threadIdx.x >= o ? (int)threadIdx.x - o : (int)threadIdx.x); }
template <typename T> T __shfl_xor_sync(unsigned, T v, int o) { return from_lane(v, (int)threadIdx.x ^ o); }
inline unsigned __ballot_sync(unsigned, bool p)
{
	unsigned m = 0;
	lane_word[threadIdx.x] = p;
	bar.arrive_and_wait();
	for (int i = 0; i < 32; ++i) m |= (unsigned)(lane_word[i] & 1) << i;
	bar.arrive_and_wait();
	return m;
}
inline int __ffs(unsigned v) { return __builtin_ffs((int)v); }
using std::max;
using std::min;
struct float4 { float x, y, z, w; };
struct uint4 { uint32_t x, y, z, w; };
inline float4 make_float4(float a, float b, float c, float d) { return {a, b, c, d}; }
inline uint4 make_uint4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) { return {a, b, c, d}; }
namespace inf {
constexpr int kWarp = 32;
enum DevErr : int { kDevKvRange = 3, kDevBadIndex = 5 };
inline void report_err(int* err, int code) { if (err && !*err) *err = code; }
inline void pdl_wait() {}
inline void pdl_trigger() {}
inline float warp_max(float x) { return x; }
inline float warp_sum(float x) { return x; }
template <typename T> struct Store;
template <typename T> void unpack_unit(const uint4&, float*, const T*);
template <typename T> uint4 pack_unit(const float*, T*);
}
"""

# reads: KT one_tile R workers min_run item_cost rows_max window n_sink G KV blk pps n_seqs, then (rows ctx) per sequence,
# then for every change: steps after which it happens (0: before begin) and (rows ctx) per sequence
MAIN = r"""
#include "k_attn_chunk.cuh"
#include <cstdio>
#include <cstdlib>
#include <thread>
#include <vector>
using namespace inf;
static int failed = 0;
#define CHECK(x) do { if (!(x)) { if (!failed) printf("%s: worker %d sequence %d from %d to %d cost %d rows %d hi %d\n", #x, w, run.s, run.from(), run.to(), run.t.cost, run.rows(), run.t.hi); failed = 1; } } while (0)

static int num() { int v; if (scanf("%d", &v) != 1) exit(3); return v; }
static std::vector<int> starts, ctx;
static void lengths(int n)
{
	int at = 0;
	for (int i = 0; i < n; ++i) {
		starts[i] = at;
		at += num();
		ctx[i] = num();
	}
	starts[n] = at;
}

template <int KT, bool kOneTile>
static void go(AttnChunkArgs a, const std::vector<int>& when, const std::vector<std::vector<int>>& then)
{
	std::vector<uint32_t> pre(a.n_seqs + 1);
	const std::vector<int> starts0 = starts, ctx0 = ctx;
	std::vector<std::vector<char>> seen; // key tiles of every item, in order
	std::vector<std::thread> lanes;
	for (int lane = 0; lane < 32; ++lane)
		lanes.emplace_back([&, lane] {
			threadIdx = {(unsigned)lane, 0};
			ac_prefix<KT>(a, pre.data());
			uint64_t tiles = 0;
			const size_t turns = when.empty() ? 1 : when.size();
			for (size_t turn = 0; turn < turns; ++turn)
				for (int w = 0; w < a.workers; ++w) {
					auto change = [&](int step) {
						__syncthreads();
						if (!when.empty() && when[turn] == step && lane == 0) {
							for (int i = 0; i <= a.n_seqs; ++i) starts[i] = then[turn][2 * i];
							for (int i = 0; i < a.n_seqs; ++i) ctx[i] = then[turn][2 * i + 1];
						}
						__syncthreads();
					};
					__syncthreads();
					if (lane == 0) starts = starts0, ctx = ctx0;
					change(0);
					AcRun<KT, kOneTile> run;
					run.begin(a, pre.data(), w);
					int steps = 0;
					const int most = a.KV * (a.n_tokens * a.G / a.R + a.n_seqs) + 1;
					while (!run.done() && steps < most) {
						if (lane == 0) {
							CHECK(0 <= run.from() && run.from() < run.to() && run.to() <= run.t.cost);
							CHECK(run.rows() >= 1 && run.rows() <= a.R);
							CHECK(run.s >= 0 && run.s < a.n_seqs && run.h >= 0 && run.h < a.KV);
							CHECK(run.q.slot >= 0 && run.q.slot < a.n_slots);
							CHECK(run.t.hi <= a.pages_per_seq * a.blk && run.t.lo >= 0);
							CHECK(ac_tile_at(run.t, run.to() - 1) * KT < max(run.t.hi, 1));
							tiles += run.to() - run.from();
							if (!run.whole() && run.from() == 0) { // what the joining kernel goes by
								ac_job(a, w, run);
								const int* j = a.jobs + (size_t)w * kAcJobInts;
								CHECK(j[kAcJobLast] >= w && j[kAcJobLast] < a.workers);
								CHECK(j[kAcJobSeq] >= 0 && j[kAcJobRow] + j[kAcJobRows] <= (a.n_tokens - j[kAcJobSeq]) * a.G);
								CHECK(j[kAcJobHead] < a.KV && j[kAcJobRows] <= a.R);
							}
						}
						change(++steps);
						run.next(a, pre.data());
					}
					if (lane == 0) CHECK(run.done());
				}
			if (lane == 0 && when.empty()) { // nothing changed: every key tile once
				uint64_t all = 0;
				for (int s = 0; s < a.n_seqs; ++s) {
					const AcSeq q = ac_seq(a, s, false);
					for (int t = 0; t * a.R < q.n * a.G; ++t) all += (uint64_t)a.KV * (ac_tile_cost<KT>(a, q, t) - a.item_cost);
				}
				if (all != tiles) { printf("%llu key tiles of %llu\n", (unsigned long long)tiles, (unsigned long long)all); failed = 1; }
			}
		});
	for (auto& t : lanes) t.join();
}

int main()
{
	AttnChunkArgs a = {};
	const int KT = num(), one = num();
	a.R = num(), a.workers = num(), a.min_run = num(), a.item_cost = num(), a.rows_max = num(), a.window = num(), a.n_sink = num(), a.G = num();
	a.KV = num(), a.blk = num(), a.pages_per_seq = num(), a.n_seqs = num();
	a.group = ac_div(a.G);
	a.H = a.G * a.KV;
	starts.resize(a.n_seqs + 1);
	ctx.resize(a.n_seqs);
	lengths(a.n_seqs);
	const std::vector<int> starts0 = starts, ctx0 = ctx;
	a.n_tokens = a.max_new = starts[a.n_seqs];
	a.n_slots = a.n_seqs;
	std::vector<int> jobs((size_t)a.workers * kAcJobInts);
	a.jobs = jobs.data();
	a.q_start = starts.data();
	a.ctx_len = ctx.data();
	std::vector<int> when;
	std::vector<std::vector<int>> then;
	for (int n = num(); n > 0; --n) {
		when.push_back(num());
		lengths(a.n_seqs);
		std::vector<int> v;
		for (int i = 0; i < a.n_seqs; ++i) v.push_back(starts[i]), v.push_back(ctx[i]);
		v.push_back(starts[a.n_seqs]);
		then.push_back(v);
	}
	starts = starts0, ctx = ctx0;
	if (KT == 16 && one) go<16, true>(a, when, then);
	else if (KT == 128) go<128, false>(a, when, then);
	else if (KT == 32) go<32, false>(a, when, then);
	else return 3;
	return failed;
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    if not shutil.which("g++"):
        pytest.skip("no g++")
    d = tmp_path_factory.mktemp("division")
    shutil.copy(os.path.join(CSRC, "k_attn_chunk.cuh"), d)
    (d / "common.cuh").write_text(STUB)
    (d / "main.cpp").write_text(MAIN)
    exe = str(d / "division")
    subprocess.run(["g++", "-std=c++20", "-O1", "-w", "-pthread", "-o", exe, str(d / "main.cpp")], check=True)
    return exe


# key tile, one tile a sequence, rows of an item, least run, an item's own cost, rows of a sequence at most
KINDS = {"rows": (16, 1, 16, 4, 0, 16), "tensor": (128, 0, 256, 4, 2, 2 ** 31 - 1), "fp32": (32, 0, 16, 2, 0, 2 ** 31 - 1)}


def run(program, kind, seqs, *, G=4, KV=2, window=0, sinks=0, workers=7, blk=16, pps=64, changes=()):
    KT, one, R, least, own, most = KINDS[kind]
    words = [KT, one, R, workers, least, own, most, window, sinks, G, KV, blk, pps, len(seqs)] + [x for s in seqs for x in s]
    words.append(len(changes))
    for step, other in changes:
        assert len(other) == len(seqs)
        words += [step] + [x for s in other for x in s]
    r = subprocess.run([program], input=" ".join(map(str, words)), text=True, capture_output=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr


def some(r, kind, n, tokens):
    """n sequences of `tokens` rows in all (the changed ones name rows of the same q)."""
    limit = 4 if kind == "rows" else 120
    rows = [r.choice([0, 1, 1, 2, r.randint(0, limit)]) for _ in range(n)]
    while sum(rows) > tokens:
        rows[r.randrange(n)] //= 2
    return [(x, r.randint(0, 1024)) for x in rows]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 4), (300, 140)])
def test_every_key_tile_has_one_worker(program, kind, window, sinks):
    r = random.Random(window)
    for n, workers in ((1, 1), (1, 9), (3, 5), (40, 16)):
        run(program, kind, [(1, 700)] + some(r, kind, n, 10 ** 6), window=window, sinks=sinks, workers=workers)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 4)])
def test_lengths_that_change_under_a_kernel(program, kind, window, sinks):
    """Sequences that are empty, shorter or longer when a worker reads them again."""
    r = random.Random(7 + window)
    seqs = [(3, 900), (1, 1000), (4, 60), (2, 700), (1, 16)] if kind == "rows" else [(300, 900), (1, 1000), (80, 90), (130, 700), (20, 16)]
    tokens = sum(n for n, _ in seqs)
    none = [(0, 0)] * 5
    changes = [(0, none), (1, none), (2, none), (0, [(n, 1) for n, _ in seqs]), (1, [(n, 2) for n, _ in seqs]),
               (0, [(1, c) for _, c in seqs]), (1, [(0, 5), (tokens if kind != "rows" else 4, 1024), (0, 0), (0, 7), (0, 1)])]
    changes += [(r.randint(0, 3), some(r, kind, 5, tokens)) for _ in range(6)]
    run(program, kind, seqs, window=window, sinks=sinks, workers=5, changes=changes)
