// Chunk attention for few rows (bf16, head_dim 64 or 128, pages a multiple of 16): sequences with at most 16
// rows per KV head, that is decode steps and a few tokens at a time.
//
// Bound by HBM: every visible K and V byte is read once.  A warp is a worker of k_attn_chunk.cuh with key tiles
// of 16 positions: it streams its run of tiles through a ring of its own (K and V of a tile per stage, one
// 5-D TMA box each, an mbarrier per stage), so nothing but its own data paces a warp, and a run goes on from
// one sequence to the next without draining the ring.  The arithmetic is warp-level mma.m16n8k16: the rows are
// the 16 rows of the A tile, S = Q.K^T with K fragments from ldmatrix, the accumulator fragments of S are the
// A fragments of P.V, V comes from ldmatrix.trans.  A warp whose run ends inside an item stores its share, which
// k_attn_chunk_combine joins with the others.
// Rounding: S, O, max and sum in fp32; P goes into the second product as two bf16 parts (rounded, then the
// rounding of what that left over: 16 bits, so that a row's error is its output's rounding), the sum adds the
// unrounded weights.  V positions that no row of the item sees are masked out of the fragments (only where such
// a tile exists: its ends).
#pragma once

#include "k_attn_chunk.cuh"
#include "tensor_core.cuh"

namespace inf {

constexpr int kCrRows = 16;
constexpr int kCrKT = 16;
constexpr int kCrWarps = 8;
constexpr int kCrThreads = kCrWarps * kWarp;

// stages of a warp's ring: 192 KB per SM over 8 warps (an SM has about 44 KB in flight at the HBM's rate and
// latency; the ring also covers the warps' unevenness)
__host__ __device__ constexpr int cr_stages(int hd) { return hd == 128 ? 3 : 6; }
__host__ __device__ constexpr uint32_t cr_tile_bytes(int hd) { return (uint32_t)kCrKT * hd * 2; } // K or V
__host__ __device__ inline size_t attn_chunk_rows_smem(int hd, int n_seqs)
{
	return 1024 + (size_t)kCrWarps * cr_stages(hd) * (2 * cr_tile_bytes(hd) + sizeof(uint64_t)) + 16 + (size_t)(n_seqs + 1) * 4;
}

// Byte offset of 16-byte chunk c (0 .. hd / 8 - 1) of position r in a tile: [8-position group][64 dims][8 x 128 bytes],
// the chunks of 128 bytes swizzled by the row as the TMA box writes them.
template <int HD>
__device__ __forceinline__ uint32_t cr_off(int r, int c)
{
	return (uint32_t)((r >> 3) * (HD / 64) * 1024 + (c >> 3) * 1024 + (r & 7) * 128 + (((c & 7) ^ (r & 7)) << 4));
}

template <int HD>
__global__ void __launch_bounds__(kCrThreads, 1)
    k_attn_chunk_rows(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const AttnChunkArgs a)
{
	constexpr int kStages = cr_stages(HD);
	constexpr uint32_t kTile = cr_tile_bytes(HD);
	extern __shared__ __align__(1024) uint8_t cr_smem[];
	uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(cr_smem) + 1023) & ~(uintptr_t)1023);
	const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
	uint8_t* ring = smem + (size_t)warp * kStages * 2 * kTile;
	uint64_t* bars = reinterpret_cast<uint64_t*>(smem + (size_t)kCrWarps * kStages * 2 * kTile) + warp * kStages;
	int* abort_s = reinterpret_cast<int*>(smem + (size_t)kCrWarps * kStages * (2 * kTile + sizeof(uint64_t)));
	uint32_t* pre = reinterpret_cast<uint32_t*>(abort_s + 4);
	volatile int* abort_flag = abort_s;
	if (threadIdx.x == 0) *abort_s = 0;
	if (lane == 0) {
		for (int i = 0; i < kStages; ++i) mbar_init(&bars[i], 1);
		mbar_fence_init();
	}
	pdl_wait();
	pdl_trigger();
	ac_prefix<kCrKT>(a, pre); // ends with a barrier
	const int worker = blockIdx.x * kCrWarps + warp;
	if (worker >= a.workers) return;
	if (lane == 0) ac_job(a, worker);
	AcRun<kCrKT, true> run, load; // where the products and where the copies are
	run.begin(a, pre, worker);
	load = run;

	// ---- the copies, kStages tiles ahead
	const uint64_t pol = policy_evict_first(); // read once
	const int blk = a.blk;
	int load_i = run.done() ? 0 : run.from(), load_to = run.done() ? 0 : run.to(), issued = 0, stage_in = 0;
	// lane j holds the page of tile ids_i + j of the item being copied: a table entry takes as long to arrive as a
	// tile's arithmetic, so they are read 32 at a time
	int ids = 0, ids_i = 0;
	auto refill = [&]() {
		ids_i = load_i;
		const int i = load_i + lane, k0 = load.done() ? 0 : ac_tile_at(load.t, i) * kCrKT;
		ids = 0; // the tile of an item that sees nothing copies some page
		if (!load.done() && i < load.to() && k0 < load.t.hi) {
			ids = a.table[(size_t)load.q.slot * a.pages_per_seq + k0 / blk];
			if (ids < 0 || ids >= a.n_pages) {
				report_err(a.status, kDevKvRange);
				ids = 0;
			}
		}
	};
	refill();
	auto fetch = [&]() { // the whole warp; no-op behind the run's end
		if (load.done()) return;
		const int page = __shfl_sync(0xFFFFFFFFu, ids, load_i - ids_i);
		const int st = __shfl_sync(0xFFFFFFFFu, stage_in, 0), head_row = __shfl_sync(0xFFFFFFFFu, load.h * blk, 0);
		const int group = blk > kCrKT ? __shfl_sync(0xFFFFFFFFu, ((ac_tile_at(load.t, load_i) * kCrKT) & (blk - 1)) >> 3, 0) : 0;
		uint8_t* dst = ring + (uint32_t)st * 2 * kTile;
		if (elect_one()) {
			mbar_arrive_expect_tx(&bars[st], 2 * kTile);
			tma_load_5d(dst, &tm_k, 0, head_row, 0, group, page, &bars[st], pol);
			tma_load_5d(dst + kTile, &tm_v, 0, head_row, 0, group, page, &bars[st], pol);
		}
		__syncwarp();
		++issued;
		if (++stage_in == kStages) stage_in = 0;
		++load_i;
		if (load_i == load_to) {
			load.next(a, pre);
			load_i = load.done() ? 0 : load.from();
			load_to = load.done() ? 0 : load.to();
			refill();
		} else if (load_i == ids_i + kWarp) {
			refill();
		}
	};
	for (int i = 0; i < kStages; ++i) fetch();

	const float sl2 = a.scale * 1.4426950408889634f; // scores in log2 units
	const int gr = lane >> 2, gc = (lane & 3) * 2;    // fragment row (and row + 8), column pair
	const int mi = lane >> 3, mr = lane & 7;          // the ldmatrix matrix and row this lane addresses
	int stage = 0;
	uint32_t phase = 0;
	bool ok = true;
	for (; ok && !run.done(); run.next(a, pre)) {
		const int rows = run.rows(), base_pos = run.q.ctx - run.q.n;
		// Q as A fragments: rows gr and gr + 8 (rows past the last one are zeros)
		uint32_t qa[HD / 16][4];
		int pos[2];
		uint64_t out_at[2];
#pragma unroll
		for (int e = 0; e < 2; ++e) {
			const int fr = min(gr + 8 * e, rows - 1);
			const int tok = a.group.div(fr), head = run.h * a.G + a.group.mod(fr);
			const bool valid = gr + 8 * e < rows;
			pos[e] = base_pos + tok;
			out_at[e] = (uint64_t)(run.q.row0 + tok) * a.out_stride + (uint64_t)head * HD;
			const uint32_t* src = reinterpret_cast<const uint32_t*>(reinterpret_cast<const bf16*>(a.q) +
			                                                        (uint64_t)(run.q.row0 + tok) * a.q_stride + (uint64_t)head * HD);
#pragma unroll
			for (int ks = 0; ks < HD / 16; ++ks) {
				qa[ks][e] = valid ? src[ks * 8 + (gc >> 1)] : 0u;
				qa[ks][2 + e] = valid ? src[ks * 8 + (gc >> 1) + 4] : 0u;
			}
		}
		const int first_pos = base_pos, last_pos = base_pos + a.group.div(rows - 1);
		float o[HD / 8][4];
#pragma unroll
		for (int i = 0; i < HD / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
		float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f}; // rows gr, gr + 8 (l: this thread's share)
		const AcTiles t = run.t;
		for (int i = run.from(); i < run.to(); ++i) {
			const int k0 = ac_tile_at(t, i) * kCrKT;
			const bool w = mbar_wait_cycles(&bars[stage], phase, abort_flag, a.status);
			ok = __all_sync(0xFFFFFFFFu, w);
			if (!ok) break;
			const uint32_t kc = smem_u32(ring + (uint32_t)stage * 2 * kTile), vc = kc + kTile;
			// S = Q.K^T, two 8-position tiles; ldmatrix x4: (tile 0, dims +0..7), (tile 0, +8..15), (tile 1, ...)
			float s[2][4];
#pragma unroll
			for (int nt = 0; nt < 2; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.0f;
#pragma unroll
			for (int ks = 0; ks < HD / 16; ++ks) {
				uint32_t b00, b01, b10, b11;
				ldsm_x4(kc + cr_off<HD>((mi >> 1) * 8 + mr, ks * 2 + (mi & 1)), b00, b01, b10, b11);
				mma_bf16_16816(s[0], qa[ks], b00, b01);
				mma_bf16_16816(s[1], qa[ks], b10, b11);
			}
			// a tile that some row does not see whole
			const bool edge = k0 + kCrKT - 1 > first_pos || (a.window && k0 <= last_pos - a.window && k0 + kCrKT > a.n_sink);
			if (edge) {
#pragma unroll
				for (int nt = 0; nt < 2; ++nt)
#pragma unroll
					for (int j = 0; j < 4; ++j)
						if (!ac_sees(a, pos[j >> 1], k0 + nt * 8 + gc + (j & 1))) s[nt][j] = -INFINITY;
			}
			float mx[2], al[2], mu[2];
#pragma unroll
			for (int e = 0; e < 2; ++e) { // the row's max over the quad (the four lanes that hold one row)
				mx[e] = fmaxf(fmaxf(s[0][2 * e], s[0][2 * e + 1]), fmaxf(s[1][2 * e], s[1][2 * e + 1])) * sl2;
				mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xFFFFFFFFu, mx[e], 1));
				mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xFFFFFFFFu, mx[e], 2));
				const float mn = fmaxf(m[e], mx[e]);
				mu[e] = mn == -INFINITY ? 0.0f : mn; // nothing seen yet: 2^(-inf) = 0
				al[e] = ex2_approx(m[e] - mu[e]);
				m[e] = mn;
			}
			float p[2][4];
#pragma unroll
			for (int nt = 0; nt < 2; ++nt)
#pragma unroll
				for (int j = 0; j < 4; ++j) p[nt][j] = ex2_approx(fmaf(s[nt][j], sl2, -mu[j >> 1]));
			uint32_t pa[4], pr[4]; // P = pa + pr: rounded, and what is left rounded again
#pragma unroll
			for (int f = 0; f < 4; ++f) {
				const float x = p[f >> 1][(f & 1) * 2], y = p[f >> 1][(f & 1) * 2 + 1];
				pa[f] = pack_bf16(x, y);
				pr[f] = pack_bf16(x - __uint_as_float(pa[f] << 16), y - __uint_as_float(pa[f] & 0xFFFF0000u));
			}
#pragma unroll
			for (int e = 0; e < 2; ++e)
				l[e] = fmaf(l[e], al[e], (p[0][2 * e] + p[0][2 * e + 1]) + (p[1][2 * e] + p[1][2 * e + 1]));
			if (__any_sync(0xFFFFFFFFu, al[0] != 1.0f || al[1] != 1.0f)) {
#pragma unroll
				for (int dt = 0; dt < HD / 8; ++dt) {
					o[dt][0] *= al[0];
					o[dt][1] *= al[0];
					o[dt][2] *= al[1];
					o[dt][3] *= al[1];
				}
			}
			// positions of the V fragments that no row of the item sees, out
			uint32_t keep0 = 0xFFFFFFFFu, keep1 = 0xFFFFFFFFu;
			if (edge) {
				auto seen = [&](int k) { return k < t.hi && (k >= t.lo || k < a.n_sink); };
				keep0 = (seen(k0 + gc) ? 0xFFFFu : 0u) | (seen(k0 + gc + 1) ? 0xFFFF0000u : 0u);
				keep1 = (seen(k0 + gc + 8) ? 0xFFFFu : 0u) | (seen(k0 + gc + 9) ? 0xFFFF0000u : 0u);
			}
			// O += P.V; ldmatrix x4 trans: (positions +0..7, dims dt), (+8..15, dt), (+0..7, dt + 1), (+8..15, dt + 1)
#pragma unroll
			for (int dt = 0; dt < HD / 8; dt += 2) {
				uint32_t b0, b1, c0, c1;
				ldsm_x4_trans(vc + cr_off<HD>((mi & 1) * 8 + mr, dt + (mi >> 1)), b0, b1, c0, c1);
				b0 &= keep0, b1 &= keep1, c0 &= keep0, c1 &= keep1;
				mma_bf16_16816(o[dt], pr, b0, b1);
				mma_bf16_16816(o[dt + 1], pr, c0, c1);
				mma_bf16_16816(o[dt], pa, b0, b1);
				mma_bf16_16816(o[dt + 1], pa, c0, c1);
			}
			__syncwarp(); // every lane is done with the stage
			fetch();
			if (++stage == kStages) {
				stage = 0;
				phase ^= 1u;
			}
		}
		if (!ok) break;
#pragma unroll
		for (int e = 0; e < 2; ++e) {
			l[e] += __shfl_xor_sync(0xFFFFFFFFu, l[e], 1);
			l[e] += __shfl_xor_sync(0xFFFFFFFFu, l[e], 2);
		}
		const bool whole = run.whole();
		float* part = a.part + (size_t)run.slot(worker) * ac_part_floats(kCrRows, HD);
#pragma unroll
		for (int e = 0; e < 2; ++e) {
			const int r = gr + 8 * e;
			if (r >= rows) continue;
			if (whole) {
				const float inv = l[e] > 0.0f ? 1.0f / l[e] : 0.0f;
				uint32_t* dst = reinterpret_cast<uint32_t*>(reinterpret_cast<bf16*>(a.out) + out_at[e]);
#pragma unroll
				for (int dt = 0; dt < HD / 8; ++dt) dst[dt * 4 + (gc >> 1)] = pack_bf16(o[dt][2 * e] * inv, o[dt][2 * e + 1] * inv);
			} else { // [hd / 4][16] float4
#pragma unroll
				for (int dt = 0; dt < HD / 8; ++dt)
					*reinterpret_cast<float2*>(part + ((size_t)(dt * 2 + (gc >> 2)) * kCrRows + r) * 4 + (gc & 3)) =
					    make_float2(o[dt][2 * e], o[dt][2 * e + 1]);
				if ((lane & 3) == 0) {
					part[(size_t)kCrRows * HD + r] = m[e];
					part[(size_t)kCrRows * HD + kCrRows + r] = l[e];
				}
			}
		}
		if (!whole && run.from() == 0 && lane == 0) ac_job(a, worker, run);
	}
	if (lane == 0) {
		// never leave the CTA with copies in flight: there are some behind a wait that ran out, or where lengths
		// changed between a copy and its products
		for (int i = max(0, issued - kStages); i < issued; ++i) {
			const long long t0 = clock64();
			while (!mbar_try_wait(&bars[i % kStages], (uint32_t)(i / kStages) & 1u))
				if (clock64() - t0 > kWaitLimitCycles) break;
		}
	}
}

} // namespace inf
