// Chunk attention on the 5th-generation tensor cores (bf16, head_dim 64 or 128, pages of 16 .. 128).
//
// A CTA is a worker of k_attn_chunk.cuh with items of 256 rows (256 / G tokens times the G heads of a KV
// group) and key tiles of 128 positions.  The rows are two subtiles of 128, each with its own softmax
// warpgroup, so that one subtile's exponentials run while the tensor cores work on the other's products:
//   warps 0-3, 4-7  a thread per row of subtile 0, 1: Q into shared memory (SWIZZLE_128B by hand), then per
//                   key tile S from tensor memory, mask, running max and sum, P = 2^(s scale - m) as bf16
//                   back into the same tensor-memory columns, in two halves; O / sum at the end
//   warps 8, 10     TMA producers of K and of V tiles into one ring (no multicast): a 5-D box per page, [8-row
//                   group][64 head dims][8 x 128 bytes], or one for the whole tile where the page ids are
//                   consecutive.  A box costs its producer about 90 cycles of issue, so that a box per page and 64
//                   head dims from one warp (32 a key tile) had paced the kernel at 4200 cycles a key tile.
//   warp 9          one thread issues S = Q.K^T (shared memory x shared memory) and O += P.V (P from
//                   tensor memory, V MN-major from shared memory)
// Tensor memory (512 columns): S0 | S1 | O0 | O1, P over the first half of its S.  The issue order
//   S0(0) S1(0) | PV0(j) S0(j+1) PV1(j) S1(j+1) | ...
// keeps S(j+1) behind the P(j) that it overwrites, and a completed S(j+1) implies a completed PV(j): O may
// then be rescaled without another wait.  That happens only when a row's max grows by more than 2^8
// (bf16 and fp32 hold the larger weights as well, and O / sum is unchanged).
// Rounding: S, O, max and sum are fp32; P is rounded to bf16 for the second product, the sum adds the
// unrounded weights (their rounding errors are independent and average out).
// Positions that no row of the item sees are not loaded page by page; where they share a page with seen
// ones, their V rows are overwritten by zeros in shared memory before the product, so that nothing they
// hold (NaN included) reaches a sum; their scores are dropped by the mask.
// Every wait is bounded; on a timeout the kernel records kDevTimeout, lets its copies and MMAs drain,
// frees tensor memory and returns.
#pragma once

#include "k_attn_chunk.cuh"
#include "tensor_core.cuh"

namespace inf {

constexpr int kCtR = 256;
constexpr int kCtKT = 128;
constexpr int kCtThreads = 384; // 3 warpgroups: softmax, softmax, (TMA, MMA, TMA, idle)
// Registers: 168 a thread at launch; the softmax warpgroups, which hold a row of 128 scores, take the third
// one's share: 2 x 208 + 88 = 3 x 168.
constexpr int kCtRegsLaunch = 168, kCtRegsSoftmax = 208, kCtRegsRest = 88;
static_assert(2 * kCtRegsSoftmax + kCtRegsRest <= 3 * kCtRegsLaunch, "register split");
constexpr int kCtMaxStages = 12;
constexpr uint32_t kCtAtom = 128 * 64 * 2; // one [128 x 64] bf16 SWIZZLE_128B block: 16 KB
constexpr float kCtRescaleLog2 = 8.0f;
constexpr int kCtPolyOf8 = 2; // of 8 pairs of weights, those whose 2^x runs on the FMA pipes

enum CtBar : int {
	kCtFull = 0,                          // [stages] TMA -> MMA (and the softmax warps, for V)
	kCtEmpty = kCtMaxStages,              // [stages] MMA done with the tile
	kCtQ = 2 * kCtMaxStages,              // [2] Q of the subtile staged (4 warps arrive)
	kCtS = kCtQ + 2,                      // [2] S ready
	kCtP = kCtS + 2,                      // [2][2] P's halves written (4 warps arrive)
	kCtO = kCtP + 4,                      // [2] the item's last product done
	kCtDrain = kCtO + 2,
	kCtBars = kCtDrain + 1
};

struct CtLayout {
	uint32_t tile, q, ring, bars, flags, pre, total;
	int stages;
};
// one K or V tile: head_dim / 64 blocks; as many ring stages as fit beside Q and the cost prefix
__host__ __device__ inline CtLayout ct_layout(int hd, int n_seqs)
{
	CtLayout L;
	L.tile = (uint32_t)(hd / 64) * kCtAtom;
	L.q = 0;
	L.ring = 2 * L.tile;
	const uint32_t rest = 304 + 16 + (uint32_t)(n_seqs + 1) * 4;
	const uint32_t room = 227 * 1024 - 1024 - rest - L.ring; // 1024: alignment of the swizzled blocks
	L.stages = (int)(room / L.tile);
	if (L.stages > kCtMaxStages) L.stages = kCtMaxStages;
	L.bars = L.ring + (uint32_t)L.stages * L.tile;
	L.flags = L.bars + 304;
	L.pre = L.flags + 16;
	L.total = 1024 + L.pre + (uint32_t)(n_seqs + 1) * 4;
	return L;
}
static_assert(kCtBars * 8 <= 304, "barriers");

// kind::f16 with A (rows x 16, two bf16 per column) in tensor memory
__device__ __forceinline__ void umma_bf16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate)
{
	asm volatile(
	    "{\n\t.reg .pred p;\n\t"
	    "setp.ne.b32 p, %4, 0;\n\t"
	    "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
	    "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
	    : "memory");
}

// ---- pairs of floats (one instruction each on sm_100) ----------------------------------
__device__ __forceinline__ uint64_t f2(float lo, float hi)
{
	uint64_t r;
	asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
	return r;
}
__device__ __forceinline__ void f2_split(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c)
{
	uint64_t r;
	asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
	return r;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b)
{
	uint64_t r;
	asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
	return r;
}
// 2^x of two values on the FMA pipes, for the share of the weights that would otherwise queue for the
// special-function unit: x = n + f with n the nearest integer (the low bits of x + 1.5 * 2^23), 2^f by the
// minimax polynomial of degree 3 on [-1/2, 1/2] (Remez exchange on the relative error: 7.5e-5 = 2^-13.7,
// against the 2^-9 of the bf16 rounding that follows), n added to the exponent.  x below -126 gives
// about 1e-38 instead of less.
__device__ __forceinline__ void ex2_poly2(uint64_t x2, float& p0, float& p1)
{
	float x0, x1;
	f2_split(x2, x0, x1);
	x2 = f2(fmaxf(x0, -126.0f), fmaxf(x1, -126.0f));
	const uint64_t t = f2_add(x2, f2(12582912.0f, 12582912.0f));
	const uint64_t n = f2_add(t, f2(-12582912.0f, -12582912.0f));
	const uint64_t f = f2_fma(n, f2(-1.0f, -1.0f), x2);
	uint64_t p = f2_fma(f, f2(0.0551716685f, 0.0551716685f), f2(0.2426111251f, 0.2426111251f));
	p = f2_fma(p, f, f2(0.6932609677f, 0.6932609677f));
	p = f2_fma(p, f, f2(0.9999280572f, 0.9999280572f));
	float t0, t1;
	f2_split(t, t0, t1);
	f2_split(p, p0, p1);
	p0 = __uint_as_float(__float_as_uint(p0) + (__float_as_uint(t0) << 23));
	p1 = __uint_as_float(__float_as_uint(p1) + (__float_as_uint(t1) << 23));
}

__device__ __forceinline__ void tmem_st_16regs(uint32_t taddr, const uint32_t (&r)[16])
{
	asm volatile(
	    "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
	    "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
	    "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
	    "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
	    : "memory");
}

// One lane of a converged warp, and a value that is the same in all of them, from lane 0: operands that the
// compiler knows to be uniform go to the tensor-core and copy instructions straight from uniform registers.
// Issued from inside a divergent branch, with operands moved over one by one, eight products took about
// 1000 cycles to issue for 512 of work.
__device__ __forceinline__ bool elect_one()
{
	uint32_t ok;
	asm volatile(
	    "{\n\t.reg .pred p;\n\t"
	    "elect.sync _|p, 0xFFFFFFFF;\n\t"
	    "selp.u32 %0, 1, 0, p;\n\t}"
	    : "=r"(ok));
	return ok != 0;
}
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __shfl_sync(0xFFFFFFFFu, v, 0); }

// the n lowest bits (none for n <= 0, all from 32 on)
__device__ __forceinline__ uint32_t low_bits(int n) { return n >= 32 ? 0xFFFFFFFFu : n <= 0 ? 0u : (1u << n) - 1u; }

// position in the ring: stage and the parity of its use
struct CtRing {
	int stage = 0;
	uint32_t phase = 0;
	__device__ __forceinline__ void next(int stages)
	{
		if (++stage == stages) {
			stage = 0;
			phase ^= 1u;
		}
	}
	__device__ __forceinline__ void skip(int n, int stages)
	{
		const int s = stage + n;
		phase ^= (uint32_t)(s / stages) & 1u;
		stage = s % stages;
	}
};

template <int HD>
__global__ void __launch_bounds__(kCtThreads, 1)
    k_attn_chunk_tc(const __grid_constant__ CUtensorMap tm_k8, const __grid_constant__ CUtensorMap tm_k1,
                    const __grid_constant__ CUtensorMap tm_v8, const __grid_constant__ CUtensorMap tm_v1, const AttnChunkArgs a)
{
	constexpr int kHalves = HD / 64;
	constexpr uint32_t kTile = (uint32_t)kHalves * kCtAtom;
	constexpr uint32_t kGroup = (uint32_t)kHalves * 1024; // 8 positions of a K or V tile: a swizzle atom per 64 head dims
	extern __shared__ __align__(1024) uint8_t ct_smem[];
	uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(ct_smem) + 1023) & ~(uintptr_t)1023);
	const CtLayout Ly = ct_layout(HD, a.n_seqs);
	const int stages = Ly.stages;
	uint8_t* q_s = smem + Ly.q;
	uint8_t* ring_s = smem + Ly.ring;
	uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Ly.bars);
	uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + Ly.flags);
	volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
	uint32_t* pre = reinterpret_cast<uint32_t*>(smem + Ly.pre);
	const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, worker = blockIdx.x;

	if (threadIdx.x == 0) {
		for (int i = 0; i < kCtBars; ++i) {
			const bool warps = (i >= kCtQ && i < kCtS) || (i >= kCtP && i < kCtO); // the four warps of a warpgroup arrive
			mbar_init(&bars[i], warps ? 4 : 1);
		}
		*abort_flag = 0;
		mbar_fence_init();
	}
	if (warp == 9) {
		asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
		asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
	}
	pdl_wait();
	pdl_trigger();
	tc_fence_before();
	ac_prefix<kCtR, kCtKT>(a, pre); // ends with a barrier
	tc_fence_after();
	const uint32_t tmem = *tmem_slot;
	AcRun<kCtR, kCtKT> run;
	run.begin(a, pre, worker);

	if (warp >= 8) {
	asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kCtRegsRest));
	if (warp == 8 || warp == 10) {
		// ---------------- TMA producers: K tiles (warp 8) and V tiles (warp 10), every other entry of the ring
		const bool is_v = warp == 10;
		const CUtensorMap* tm8 = is_v ? &tm_v8 : &tm_k8;
		const CUtensorMap* tm1 = is_v ? &tm_v1 : &tm_k1;
		const uint64_t pol = policy_evict_normal();
		const int blk = a.blk, pages = kCtKT / blk;
		CtRing r;
		if (is_v) r.next(stages);
		uint32_t entry = is_v ? 1u : 0u; // entries of the ring before this one
		bool ok = true;
		for (; ok && !run.done(); run.next(a, pre)) {
			const int* bt = a.table + (size_t)run.q.slot * a.pages_per_seq;
			const int hi = run.t.hi, lo = run.t.lo, sinks = min(a.n_sink, hi);
			// lane p holds page p of the tile; pages that no row sees stay out.  The next tile's ids are read
			// before this one's stage is waited for.
			auto sees = [&](int i) {
				const int kp = ac_tile_at(run.t, i) * kCtKT + lane * blk;
				return lane < pages && kp < hi && (kp + blk > lo || kp < sinks);
			};
			auto look = [&](int i) { return sees(i) ? bt[ac_tile_at(run.t, i) * pages + lane] : 0; };
			int ahead = look(run.from());
			for (int i = run.from(); ok && i < run.to(); ++i) {
				const bool seen = sees(i);
				int page = ahead;
				ahead = i + 1 < run.to() ? look(i + 1) : 0;
				if (seen && (page < 0 || page >= a.n_pages)) {
					report_err(a.status, kDevKvRange);
					page = 0;
				}
				const unsigned mask = __ballot_sync(0xFFFFFFFFu, seen);
				const int page0 = __shfl_sync(0xFFFFFFFFu, page, 0);
				const bool one_box = mask == (1u << pages) - 1u && __all_sync(0xFFFFFFFFu, lane >= pages || page == page0 + lane);
				const uint32_t bytes = (uint32_t)__popc(mask) * (uint32_t)blk * HD * 2;
				if (entry >= (uint32_t)stages) {
					const bool w = mbar_wait_cycles(&bars[kCtEmpty + r.stage], r.phase ^ 1u, abort_flag, a.status);
					ok = __all_sync(0xFFFFFFFFu, w);
					if (!ok) break;
				}
				const uint32_t stage = uniform((uint32_t)r.stage);
				uint8_t* dst = ring_s + stage * kTile;
				uint64_t* full = &bars[kCtFull + stage];
				const int head_row = (int)uniform((uint32_t)(run.h * blk));
				if (elect_one()) {
					if (bytes) mbar_arrive_expect_tx(full, bytes);
					else mbar_arrive(full);
				}
				__syncwarp();
				if (one_box) {
					if (elect_one()) tma_load_5d(dst, tm8, 0, head_row, 0, 0, page0, full, pol);
				} else {
#pragma unroll
					for (int p = 0; p < kCtKT / 16; ++p) {
						const int id = __shfl_sync(0xFFFFFFFFu, page, p);
						if (((mask >> p) & 1u) && elect_one()) tma_load_5d(dst + (uint32_t)(p * blk) * HD * 2, tm1, 0, head_row, 0, 0, id, full, pol);
					}
				}
				entry += 2;
				r.skip(2, stages);
			}
		}
		if (!ok) {
			// never leave the CTA with copies in flight: this producer's last entries
			__syncwarp();
			CtRing back;
			if (is_v) back.next(stages);
			for (uint32_t i = is_v ? 1u : 0u; i < entry; i += 2, back.skip(2, stages)) {
				if (i + (uint32_t)stages < entry) continue;
				const uint64_t t0 = global_timer_ns();
				while (!mbar_try_wait(&bars[kCtFull + back.stage], back.phase))
					if (global_timer_ns() - t0 > kWaitLimitNs) break;
			}
		}
	} else if (warp == 9) {
		// ---------------- MMA issuer: the warp runs the pipeline converged, one elected lane issues
		constexpr uint32_t idesc_s = umma_idesc_bf16(128, kCtKT);
		constexpr uint32_t idesc_o = umma_idesc_bf16(128, HD) | (1u << 16); // B (V) MN-major
		const uint32_t qa = smem_u32(q_s), ra = smem_u32(ring_s), tm = uniform(tmem);
		CtRing r;
		uint32_t q_par[2] = {0, 0}, p_par[2] = {0, 0};
		auto wait = [&](int bar, uint32_t par) {
			const bool w = mbar_wait_cycles(&bars[bar], par, abort_flag, a.status);
			return (bool)__all_sync(0xFFFFFFFFu, w);
		};
		auto commit = [&](int bar) {
			if (elect_one()) umma_commit(&bars[bar]);
			__syncwarp();
		};
		auto issue_s = [&](int sub, uint32_t stage) {
			const uint64_t da = umma_desc_sw128(qa + (uint32_t)sub * kTile);
			const uint64_t db = umma_desc_sw128_lbo(ra + stage * kTile, 16, kGroup);
			if (elect_one()) {
#pragma unroll
				for (int k = 0; k < HD / 16; ++k)
					umma_bf16(tm + (uint32_t)sub * kCtKT, da + (uint32_t)((k >> 2) * (kCtAtom / 16) + (k & 3) * 2),
					          db + (uint32_t)((k >> 2) * 64 + (k & 3) * 2), idesc_s, k > 0 ? 1u : 0u);
				umma_commit(&bars[kCtS + sub]);
			}
			__syncwarp();
		};
		auto issue_pv = [&](int sub, uint32_t stage, uint32_t acc) -> bool {
			const uint64_t dv = umma_desc_sw128_lbo(ra + stage * kTile, 1024, kGroup);
			const uint32_t pa = tm + (uint32_t)sub * kCtKT, od = tm + 2 * kCtKT + (uint32_t)(sub * HD);
#pragma unroll
			for (int half = 0; half < 2; ++half) {
				if (!wait(kCtP + sub * 2 + half, p_par[sub])) return false;
				tc_fence_after();
				if (elect_one()) {
#pragma unroll
					for (int k = half * 4; k < half * 4 + 4; ++k)
						umma_bf16_ts(od, pa + (uint32_t)k * 8, dv + (uint32_t)(k * 2 * kGroup / 16), idesc_o, k > 0 ? 1u : acc);
				}
				__syncwarp();
			}
			p_par[sub] ^= 1u;
			return true;
		};
		bool ok = true;
		for (; ok && !run.done(); run.next(a, pre)) {
			const int n = run.to() - run.from();
			const bool two = run.rows() > 128;
			// K of the first tile
			ok = wait(kCtFull + r.stage, r.phase) && wait(kCtQ, q_par[0]);
			if (!ok) break;
			q_par[0] ^= 1u;
			tc_fence_after();
			uint32_t ks = uniform((uint32_t)r.stage);
			issue_s(0, ks);
			if (two) {
				ok = wait(kCtQ + 1, q_par[1]);
				if (!ok) break;
				q_par[1] ^= 1u;
				tc_fence_after();
				issue_s(1, ks);
			}
			commit(kCtEmpty + (int)ks);
			r.next(stages);
			for (int j = 0; ok && j < n; ++j) {
				const uint32_t vs = uniform((uint32_t)r.stage);
				ok = wait(kCtFull + (int)vs, r.phase);
				if (!ok) break;
				r.next(stages);
				ok = issue_pv(0, vs, j > 0 ? 1u : 0u);
				if (!ok) break;
				ks = uniform((uint32_t)r.stage);
				if (j + 1 < n) {
					ok = wait(kCtFull + (int)ks, r.phase);
					if (!ok) break;
					tc_fence_after();
					issue_s(0, ks);
				} else {
					commit(kCtO);
				}
				if (two) {
					ok = issue_pv(1, vs, j > 0 ? 1u : 0u);
					if (!ok) break;
				}
				commit(kCtEmpty + (int)vs);
				if (j + 1 < n) {
					if (two) issue_s(1, ks);
					commit(kCtEmpty + (int)ks);
					r.next(stages);
				} else if (two) {
					commit(kCtO + 1);
				}
			}
		}
		// every product is done before tensor memory is freed, whatever ended the loop
		commit(kCtDrain);
		const long long t0 = clock64();
		while (!mbar_try_wait(&bars[kCtDrain], 0))
			if (clock64() - t0 > kWaitLimitCycles) break;
		__syncwarp();
	}
	} else {
		asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kCtRegsSoftmax));
		// ---------------- softmax: subtile `sub`, a thread per row
		const int sub = warp >> 2, quarter = warp & 3;
		const int r = quarter * 32 + lane;
		const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
		const uint32_t ts = tmem + (uint32_t)sub * kCtKT + lanes, to = tmem + 2 * kCtKT + (uint32_t)(sub * HD) + lanes;
		uint8_t* qd = q_s + (size_t)sub * kTile;
		const float sl2 = a.scale * 1.4426950408889634f; // scores in log2 units
		CtRing ring;
		uint32_t s_par = 0, o_par = 0;
		bool ok = true;
		// waits are voted warp-wide so that the warp stays converged for tcgen05.ld / st
		auto wait = [&](int bar, uint32_t par) {
			const bool w = mbar_wait_cycles(&bars[bar], par, abort_flag, a.status);
			return (bool)__all_sync(0xFFFFFFFFu, w);
		};
		if (warp == 0 && lane == 0) ac_job<kCtR, kCtKT>(a, worker, nullptr);
		for (; ok && !run.done(); run.next(a, pre)) {
			const int from = run.from(), to_tile = run.to();
			const int valid = min(128, run.rows() - sub * 128); // rows of this subtile
			if (warp == 0 && lane == 0 && from == 0 && !run.whole()) ac_job<kCtR, kCtKT>(a, worker, &run);
			if (valid <= 0) {
				ring.skip(2 * (to_tile - from), stages);
				continue;
			}
			// rows past the last one repeat it: their scores are masked alike, their outputs not stored
			const int fr = run.tile * kCtR + sub * 128 + min(r, valid - 1);
			const int tok = a.group.div(fr), head = run.h * a.G + a.group.mod(fr);
			const int pos = run.q.ctx - run.q.n + tok;
			{
				// Q: the warp reads its rows one after the other, 16 bytes per lane, all in flight together
				const uint64_t src = (uint64_t)(run.q.row0 + tok) * a.q_stride + (uint64_t)head * HD;
				constexpr int kUnits = HD / 8, kPer = 32 / kUnits; // 16-byte units of a row, rows per step
				const int c = lane % kUnits;
				uint4 u[32 / kPer];
#pragma unroll
				for (int i = 0; i < 32 / kPer; ++i) {
					const uint64_t s = __shfl_sync(0xFFFFFFFFu, src, i * kPer + lane / kUnits);
					u[i] = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const bf16*>(a.q) + s + c * 8));
				}
#pragma unroll
				for (int i = 0; i < 32 / kPer; ++i)
					*reinterpret_cast<uint4*>(qd + (size_t)(c >> 3) * kCtAtom + sw128_off(quarter * 32 + i * kPer + lane / kUnits, c & 7)) = u[i];
				asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
				__syncwarp();
				if (lane == 0) mbar_arrive(&bars[kCtQ + sub]);
			}
			const int lo = run.t.lo, hi = run.t.hi;
			float m = -INFINITY, l = 0.0f;
			for (int i = from; i < to_tile; ++i) {
				const int k0 = ac_tile_at(run.t, i) * kCtKT;
				ring.next(stages); // past K
				const int vstage = ring.stage;
				const uint32_t vphase = ring.phase;
				ring.next(stages);
				ok = wait(kCtS + sub, s_par);
				if (!ok) break;
				s_par ^= 1u;
				tc_fence_after();
				float v[kCtKT];
#pragma unroll
				for (int c = 0; c < kCtKT; c += 32) tmem_ld_32cols_nowait(ts + (uint32_t)c, v + c);
				asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
				// V rows that no row of the item sees become zeros
				if (k0 + kCtKT > hi || (k0 < lo && min(k0 + kCtKT, lo) > a.n_sink)) {
					ok = wait(kCtFull + vstage, vphase);
					if (!ok) break;
					const int k = k0 + r;
					if (k >= hi || (k < lo && k >= a.n_sink)) {
						uint4* row = reinterpret_cast<uint4*>(ring_s + (size_t)vstage * kTile + (r >> 3) * kGroup + (r & 7) * 128);
#pragma unroll
						for (int h = 0; h < kHalves; ++h)
#pragma unroll
							for (int c = 0; c < 8; ++c) row[h * 64 + c] = make_uint4(0, 0, 0, 0);
					}
					asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
				}
				// mask: keys above `top` and, under a window, those from the sinks to below `bot`
				const int top = pos - k0, bot = a.window ? pos - a.window + 1 - k0 : 0, sk = a.n_sink - k0;
				if (__any_sync(0xFFFFFFFFu, top < kCtKT - 1 || (bot > 0 && sk < kCtKT))) {
#pragma unroll
					for (int q = 0; q < 4; ++q) {
						// a bit per key; tested with constants, so that no lane branches
						const uint32_t w = low_bits(top + 1 - q * 32) & (~low_bits(bot - q * 32) | low_bits(sk - q * 32));
#pragma unroll
						for (int c = 0; c < 32; ++c) v[q * 32 + c] = (w & (1u << c)) ? v[q * 32 + c] : -INFINITY;
					}
				}
				float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
				for (int c = 0; c < kCtKT; ++c) m4[c & 3] = fmaxf(m4[c & 3], v[c]);
				const float mt = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * sl2;
				const bool grow = mt > m + kCtRescaleLog2 || (m == -INFINITY && mt != -INFINITY);
				const float mn = grow ? mt : m;
				if (i > from && __any_sync(0xFFFFFFFFu, grow && m != -INFINITY)) {
					// S is complete, so every earlier product is: O holds still
					const float f = grow && m != -INFINITY ? ex2_approx(m - mn) : 1.0f;
					l *= f;
#pragma unroll 1
					for (int c = 0; c < HD; c += 32) {
						float o[32];
						tmem_ld_32cols(to + (uint32_t)c, o);
#pragma unroll
						for (int k = 0; k < 32; ++k) o[k] *= f;
						tmem_st_32cols(to + (uint32_t)c, o);
					}
				}
				m = mn;
				const float mu = m == -INFINITY ? 0.0f : m; // nothing seen yet: 2^(-inf) = 0
				const uint64_t sl2x2 = f2(sl2, sl2), mux2 = f2(-mu, -mu);
				uint64_t sum[2] = {0, 0};
#pragma unroll
				for (int q = 0; q < 4; ++q) {
					uint32_t pk[16];
#pragma unroll
					for (int c = 0; c < 16; ++c) {
						const uint64_t x = f2_fma(f2(v[q * 32 + 2 * c], v[q * 32 + 2 * c + 1]), sl2x2, mux2);
						float p0, p1;
						if (c % 8 < kCtPolyOf8) {
							ex2_poly2(x, p0, p1);
						} else {
							f2_split(x, p0, p1);
							p0 = ex2_approx(p0);
							p1 = ex2_approx(p1);
						}
						sum[c & 1] = f2_add(sum[c & 1], f2(p0, p1));
						pk[c] = pack_bf16(p0, p1);
					}
					tmem_st_16regs(ts + (uint32_t)q * 16, pk);
					if (q & 1) {
						asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
						tc_fence_before();
						__syncwarp();
						if (lane == 0) mbar_arrive(&bars[kCtP + sub * 2 + (q >> 1)]);
					}
				}
				float s0, s1;
				f2_split(f2_add(sum[0], sum[1]), s0, s1);
				l += s0 + s1;
			}
			if (!ok) break;
			ok = wait(kCtO + sub, o_par);
			if (!ok) break;
			o_par ^= 1u;
			tc_fence_after();
			float o[HD];
#pragma unroll
			for (int c = 0; c < HD; c += 32) tmem_ld_32cols_nowait(to + (uint32_t)c, o + c);
			asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
			// a row that has seen nothing: its weights were 2^-126 at most, of whatever V holds
			if (m == -INFINITY) l = 0.0f;
			if (run.whole()) {
				const float inv = l > 0.0f ? 1.0f / l : 0.0f;
				uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<bf16*>(a.out) + (uint64_t)(run.q.row0 + tok) * a.out_stride +
				                                      (uint64_t)head * HD);
				if (r < valid) {
#pragma unroll
					for (int u = 0; u < HD / 8; ++u)
						dst[u] = make_uint4(pack_bf16(o[8 * u] * inv, o[8 * u + 1] * inv), pack_bf16(o[8 * u + 2] * inv, o[8 * u + 3] * inv),
						                    pack_bf16(o[8 * u + 4] * inv, o[8 * u + 5] * inv), pack_bf16(o[8 * u + 6] * inv, o[8 * u + 7] * inv));
				}
			} else if (r < valid) {
				// a share of a divided item: [hd / 4][256] float4, so that a warp's stores are whole lines
				float* part = a.part + (size_t)run.slot(worker) * ac_part_floats(kCtR, HD);
				const int pr = sub * 128 + r;
#pragma unroll
				for (int u = 0; u < HD / 4; ++u)
					reinterpret_cast<float4*>(part)[(size_t)u * kCtR + pr] = make_float4(o[4 * u], o[4 * u + 1], o[4 * u + 2], o[4 * u + 3]);
				part[(size_t)kCtR * HD + pr] = m;
				part[(size_t)kCtR * HD + kCtR + pr] = l;
			}
			tc_fence_before(); // the next item's first product overwrites O after this warpgroup's next P
		}
	}
	tc_fence_before();
	__syncthreads();
	if (warp == 9) {
		tc_fence_after();
		asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
	}
}

} // namespace inf
