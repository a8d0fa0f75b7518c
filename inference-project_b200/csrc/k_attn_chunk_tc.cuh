// Chunk attention on the 5th-generation tensor cores (bf16, head_dim 64 or 128, pages of 16 .. 128).
//
// A CTA is a worker of k_attn_chunk.cuh with items of up to 256 rows (2 floor(128 / G) tokens times the G
// heads of a KV group) and key tiles of 128 positions.  The rows are two subtiles of up to 128, each with its
// own warpgroup, so that one subtile's exponentials run while the tensor cores work on the other's products:
//   warps 0-3, 4-7  a thread per row of subtile 0, 1: per key tile S from tensor memory into registers, mask,
//                   running max, P = 2^(s scale - m) as bf16 back into the same tensor-memory columns, then
//                   the row's sum (off the path to the next product); O / sum at the end
//   warps 8, 10     TMA producers of K and of V tiles into one ring (no multicast): a 5-D box per page, [8-row
//                   group][64 head dims][8 x 128 bytes], or one for the whole tile where the page ids are
//                   consecutive
//   warp 9          issues S = Q.K^T (shared memory x shared memory) and O += P.V (P from tensor memory, V
//                   MN-major from shared memory)
//   warp 11         TMA producer of Q: a box of floor(128 / G) tokens x G heads per subtile and 64 head dims
// Tensor memory (512 columns): S0 | S1 | O0 | O1, P over the first half of its S.  The issue order
//   S0(0) S1(0) | PV0(j) S0(j+1) PV1(j) S1(j+1) | ...
// keeps S(j+1) behind the P(j) that it overwrites, keeps the subtiles half a period apart (when each
// warpgroup issued its own products both waited and both computed at the same time), and makes a completed
// S(j+1) imply a completed PV(j): O may then be rescaled without another wait.  That happens only when a
// row's max grows by more than 2^8 (bf16 and fp32 hold the larger weights as well, and O / sum is unchanged).
// Rounding: S, O, max and sum are fp32; P is rounded to bf16 for the second product, as in the library's prefill
// attention, the sum adds the unrounded weights.  The weights' roundings are independent of each other and add
// about as much to a row's error as the output's own (root mean square 0.0023 of the outputs, 0.0017 with exact
// weights); a second bf16 part, which the row kernel has, would double P.V on the tensor pipe here.
// Positions that no row of the item sees are not loaded page by page; where they share a page with seen
// ones, their V rows are overwritten by zeros in shared memory before the product, so that nothing they
// hold (NaN included) reaches a sum; their scores are dropped by the mask.
// Every wait is bounded; on a timeout the kernel records kDevTimeout, lets its copies and MMAs drain,
// frees tensor memory and returns.
#pragma once

#include "k_attn_chunk.cuh"
#include "tensor_core.cuh"

namespace inf {

constexpr int kCtRows = 128; // rows of a subtile at most: floor(128 / G) tokens times G heads
constexpr int kCtKT = 128;   // keys of a tile
constexpr int kCtThreads = 384; // 3 warpgroups: subtile 0, subtile 1, copies and products
// Registers: 168 a thread at launch; the softmax warpgroups, which hold a row of 128 scores, take of the third
// one's share: 2 x 184 + 136 = 3 x 168, the split in which no role spills.
constexpr int kCtRegsLaunch = 168, kCtRegsSoftmax = 184, kCtRegsRest = 136;
static_assert(2 * kCtRegsSoftmax + kCtRegsRest <= 3 * kCtRegsLaunch, "register split");
constexpr int kCtMaxStages = 12;
constexpr uint32_t kCtAtom = 128 * 64 * 2; // one [128 x 64] bf16 SWIZZLE_128B block: 16 KB
constexpr float kCtRescaleLog2 = 8.0f;  // growth of a row's max that O is not rescaled for
// An item costs about 2 key tiles beside its own (its masked tiles, its last product's wait, its output): without
// it the worker that met 16 items of a short prompt ended 30 us behind the others (8 chunks beside 24 decodes).
constexpr int kCtItemCost = 2;
constexpr uint32_t kCtBarBytes = 304;

enum CtBar : int {
	kCtFull = 0,                          // [stages] tile in the ring
	kCtEmpty = kCtMaxStages,              // [stages] both subtiles' products done with it
	kCtQ = 2 * kCtMaxStages,              // [2] Q of the subtile loaded
	kCtQFree = kCtQ + 2,                  // [2] the item's last S done with it
	kCtS = kCtQFree + 2,                  // [2] S ready
	kCtP = kCtS + 2,                      // [2] P written (4 warps arrive)
	kCtO = kCtP + 2,                      // [2] the item's last product done
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
	const uint32_t rest = kCtBarBytes + 16 + (uint32_t)(n_seqs + 1) * 4;
	const uint32_t room = 227 * 1024 - 1024 - rest - L.ring; // 1024: alignment of the swizzled blocks
	L.stages = (int)(room / L.tile);
	if (L.stages > kCtMaxStages) L.stages = kCtMaxStages;
	L.bars = L.ring + (uint32_t)L.stages * L.tile;
	L.flags = L.bars + kCtBarBytes;
	L.pre = L.flags + 16;
	L.total = 1024 + L.pre + (uint32_t)(n_seqs + 1) * 4;
	return L;
}
static_assert(kCtBars * 8 <= kCtBarBytes, "barriers");

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

__device__ __forceinline__ void tmem_st_16regs(uint32_t taddr, const uint32_t (&r)[16])
{
	asm volatile(
	    "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
	    "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
	    "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
	    "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
	    : "memory");
}

// the n lowest bits (none for n <= 0, all from 32 on)
__device__ __forceinline__ uint32_t low_bits(int n) { return n >= 32 ? 0xFFFFFFFFu : n <= 0 ? 0u : (1u << n) - 1u; }

// 32 columns without the wait; the registers hold the values only behind tmem_ld_wait, which ties them to it
__device__ __forceinline__ void tmem_ld_32(uint32_t taddr, float (&v)[32])
{
	asm volatile(
	    "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
	    "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
	    "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
	    : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
	      "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]),
	      "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]),
	      "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
	    : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld_wait(float (&v)[32])
{
	asm volatile("tcgen05.wait::ld.sync.aligned;"
	             : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]),
	               "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]), "+f"(v[16]),
	               "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]), "+f"(v[23]), "+f"(v[24]),
	               "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29])
	             :
	             : "memory");
	asm volatile("" : "+f"(v[30]), "+f"(v[31]));
}

// 16 columns of O times f (a row each lane), in few registers: it runs while a row of scores is held
__device__ __forceinline__ void tmem_scale_16(uint32_t taddr, float f)
{
	float v[16];
	asm volatile(
	    "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
	    "tcgen05.wait::ld.sync.aligned;"
	    : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
	      "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
	    : "r"(taddr)
	    : "memory");
	uint32_t w[16];
#pragma unroll
	for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(v[i] * f);
	tmem_st_16regs(taddr, w);
	asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

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
    k_attn_chunk_tc(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k8, const __grid_constant__ CUtensorMap tm_k1,
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
		for (int i = 0; i < kCtBars; ++i) mbar_init(&bars[i], i >= kCtP && i < kCtO ? 4 : 1);
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
	ac_prefix<kCtKT>(a, pre); // ends with a barrier
	tc_fence_after();
	const uint32_t tmem = *tmem_slot;

	if (warp >= 8) {
		asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kCtRegsRest));
		AcRun<kCtKT> run; // begun behind setmaxnreg: state held across it spills
		run.begin(a, pre, worker);
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
						const bool w = mbar_wait_cycles<64>(&bars[kCtEmpty + r.stage], r.phase ^ 1u, abort_flag, a.status);
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
			// never leave the CTA with copies in flight (there are some behind a wait that ran out, or where lengths
			// changed between a copy and its products): this producer's last entries
			__syncwarp();
			for (uint32_t back = 2; back <= (uint32_t)stages && back <= entry; back += 2) {
				const uint32_t i = entry - back, use = i / (uint32_t)stages;
				const uint64_t t0 = global_timer_ns();
				while (!mbar_try_wait(&bars[kCtFull + (i - use * (uint32_t)stages)], use & 1u))
					if (global_timer_ns() - t0 > kWaitLimitNs) break;
			}
		} else if (warp == 9) {
			// ---------------- product issuer: the warp runs the pipeline converged, one elected lane issues
			constexpr uint32_t idesc_s = umma_idesc_bf16(128, kCtKT);
			constexpr uint32_t idesc_o = umma_idesc_bf16(128, HD) | (1u << 16); // B (V) MN-major
			const uint32_t qa = smem_u32(q_s), ra = smem_u32(ring_s), tm = uniform(tmem);
			CtRing r;
			uint32_t q_par[2] = {0, 0}, p_par[2] = {0, 0};
			auto wait = [&](int bar, uint32_t par) {
				const bool w = mbar_wait_cycles(&bars[bar], par, abort_flag, a.status);
				return (bool)__all_sync(0xFFFFFFFFu, w);
			};
			auto mma_s = [&](int sub, uint32_t stage) { // by the elected lane
				const uint64_t da = umma_desc_sw128(qa + (uint32_t)sub * kTile);
				const uint64_t db = umma_desc_sw128_lbo(ra + stage * kTile, 16, kGroup);
#pragma unroll
				for (int k = 0; k < HD / 16; ++k)
					umma_bf16(tm + (uint32_t)sub * kCtKT, da + (uint32_t)((k >> 2) * (kCtAtom / 16) + (k & 3) * 2),
					          db + (uint32_t)((k >> 2) * 64 + (k & 3) * 2), idesc_s, k > 0 ? 1u : 0u);
				umma_commit(&bars[kCtS + sub]);
			};
			auto mma_pv = [&](int sub, uint32_t stage, uint32_t acc) {
				const uint64_t dv = umma_desc_sw128_lbo(ra + stage * kTile, 1024, kGroup);
				const uint32_t pa = tm + (uint32_t)sub * kCtKT, od = tm + 2 * kCtKT + (uint32_t)(sub * HD);
#pragma unroll
				for (int k = 0; k < kCtKT / 16; ++k)
					umma_bf16_ts(od, pa + (uint32_t)k * 8, dv + (uint32_t)(k * 2 * kGroup / 16), idesc_o, k > 0 ? 1u : acc);
			};
			bool ok = true, busy = !run.done();
			int n = busy ? run.to() - run.from() : 0, subs = busy && run.rows() > (a.R >> 1) ? 2 : 1;
			while (ok && busy) {
				// S of the first tile
				uint32_t ks = uniform((uint32_t)r.stage);
				ok = wait(kCtFull + (int)ks, r.phase);
#pragma unroll
				for (int sub = 0; sub < 2; ++sub) {
					if (!ok || sub >= subs) break;
					ok = wait(kCtQ + sub, q_par[sub]);
					if (!ok) break;
					q_par[sub] ^= 1u;
					tc_fence_after();
					if (elect_one()) {
						mma_s(sub, ks);
						if (n == 1) umma_commit(&bars[kCtQFree + sub]);
						if (sub == subs - 1) umma_commit(&bars[kCtEmpty + ks]);
					}
					__syncwarp();
				}
				if (!ok) break;
				r.next(stages);
				// the next item, found while the softmax warps work
				run.next(a, pre);
				busy = !run.done();
				const int next_n = busy ? run.to() - run.from() : 0, next_subs = busy && run.rows() > (a.R >> 1) ? 2 : 1;
				for (int j = 0; ok && j < n; ++j) {
					// V of this tile and K of the next are waited for ahead of P, so that nothing but the issue
					// stands between P and the next S
					const uint32_t vs = uniform((uint32_t)r.stage);
					ok = wait(kCtFull + (int)vs, r.phase);
					if (!ok) break;
					r.next(stages);
					const bool more = j + 1 < n, last_s = j + 2 == n;
					if (more) {
						ks = uniform((uint32_t)r.stage);
						ok = wait(kCtFull + (int)ks, r.phase);
						if (!ok) break;
						r.next(stages);
					}
					const uint32_t acc = j > 0 ? 1u : 0u;
#pragma unroll
					for (int sub = 0; sub < 2; ++sub) {
						if (!ok || sub >= subs) break;
						ok = wait(kCtP + sub, p_par[sub]);
						if (!ok) break;
						p_par[sub] ^= 1u;
						tc_fence_after();
						if (elect_one()) {
							mma_pv(sub, vs, acc);
							if (more) {
								mma_s(sub, ks);
								if (last_s) umma_commit(&bars[kCtQFree + sub]);
							} else {
								umma_commit(&bars[kCtO + sub]);
							}
							if (sub == subs - 1) {
								umma_commit(&bars[kCtEmpty + vs]);
								if (more) umma_commit(&bars[kCtEmpty + ks]);
							}
						}
						__syncwarp();
					}
				}
				n = next_n;
				subs = next_subs;
			}
			// every product is done before tensor memory is freed, whatever ended the loop
			if (elect_one()) umma_commit(&bars[kCtDrain]);
			__syncwarp();
			const long long t0 = clock64();
			while (!mbar_try_wait(&bars[kCtDrain], 0))
				if (clock64() - t0 > kWaitLimitCycles) break;
			__syncwarp();
		} else {
			// ---------------- TMA producer of Q: both subtiles of the next item while the last one finishes
			const uint32_t bytes = (uint32_t)(a.R >> 1) * HD * 2;
			const int toks = a.group.div(a.R >> 1); // tokens of a subtile
			const uint64_t pol = policy_evict_first();
			uint32_t uses[2] = {0, 0};
			bool ok = true;
			for (; ok && !run.done(); run.next(a, pre)) {
				const int subs = run.rows() > (a.R >> 1) ? 2 : 1;
				const int head = (int)uniform((uint32_t)(run.h * a.G)), tok = (int)uniform((uint32_t)(run.q.row0 + run.tile * 2 * toks));
#pragma unroll
				for (int sub = 0; sub < 2; ++sub) {
					if (!ok || sub >= subs) break;
					if (uses[sub] > 0) {
						const bool w = mbar_wait_cycles<500>(&bars[kCtQFree + sub], (uses[sub] - 1) & 1u, abort_flag, a.status);
						ok = __all_sync(0xFFFFFFFFu, w);
						if (!ok) break;
					}
					if (elect_one()) {
						mbar_arrive_expect_tx(&bars[kCtQ + sub], bytes);
#pragma unroll
						for (int h = 0; h < kHalves; ++h)
							tma_load_3d(q_s + (uint32_t)sub * kTile + h * kCtAtom, &tm_q, h * 64, head, tok + sub * toks, &bars[kCtQ + sub], pol);
					}
					__syncwarp();
					++uses[sub];
				}
			}
			for (int sub = 0; sub < 2; ++sub) { // copies in flight
				if (uses[sub] == 0) continue;
				const long long t0 = clock64();
				while (!mbar_try_wait(&bars[kCtQ + sub], (uses[sub] - 1) & 1u))
					if (clock64() - t0 > kWaitLimitCycles) break;
			}
		}
	} else {
		asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kCtRegsSoftmax));
		AcRun<kCtKT> run;
		run.begin(a, pre, worker);
		// ---------------- softmax: subtile `sub`, a thread per row
		const int sub = warp >> 2, quarter = warp & 3;
		const int r = quarter * 32 + lane, half_rows = a.R >> 1;
		const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
		const uint32_t ts = tmem + (uint32_t)sub * kCtKT + lanes, to = tmem + 2 * kCtKT + (uint32_t)(sub * HD) + lanes;
		const float sl2 = a.scale * 1.4426950408889634f; // scores in log2 units
		const uint64_t sl2x2 = f2(sl2, sl2);
		const int n_sink = a.n_sink;
		CtRing ring;
		uint32_t s_par = 0, o_par = 0;
		bool ok = true;
		// waits are voted warp-wide so that the warp stays converged for tcgen05.ld / st
		auto wait = [&](int bar, uint32_t par) {
			const bool w = mbar_wait_cycles(&bars[bar], par, abort_flag, a.status);
			return (bool)__all_sync(0xFFFFFFFFu, w);
		};
		if (warp == 0 && lane == 0) ac_job(a, worker);
		while (ok && !run.done()) {
			const int from = run.from(), to_tile = run.to();
			const int valid = min(half_rows, run.rows() - sub * half_rows); // rows of this subtile
			if (warp == 0 && lane == 0 && from == 0 && !run.whole()) ac_job(a, worker, run);
			if (valid <= 0) {
				ring.skip(2 * (to_tile - from), stages);
				run.next(a, pre);
				continue;
			}
			// rows past the last one repeat its position: their scores are masked alike, their outputs not stored
			const int fr = run.tile * a.R + sub * half_rows + min(r, valid - 1);
			const int tok = a.group.div(fr), head = run.h * a.G + a.group.mod(fr);
			const int pos = run.q.ctx - run.q.n + tok;
			const int lo = run.t.lo, hi = run.t.hi;
			const int bot0 = a.window ? pos - a.window + 1 : 0; // the row's window (0: from the start)
			float m = -INFINITY, l = 0.0f;
			for (int i = from; i < to_tile; ++i) {
				const int k0 = ac_tile_at(run.t, i) * kCtKT;
				ring.next(stages); // past K
				const int vstage = ring.stage;
				const uint32_t vphase = ring.phase;
				ring.next(stages);
				// visible keys, a bit each: up to `top` and, under a window, from `bot` on or below the sinks' end
				const int top = pos - k0, bot = bot0 - k0, sk = n_sink - k0;
				const bool masked = __any_sync(0xFFFFFFFFu, top < kCtKT - 1 || (bot > 0 && sk < kCtKT));
				const bool ragged = k0 + kCtKT > hi || (k0 < lo && min(k0 + kCtKT, lo) > n_sink);
				ok = wait(kCtS + sub, s_par);
				if (__builtin_expect(!ok, 0)) break;
				s_par ^= 1u;
				tc_fence_after();
				float v[4][32];
#pragma unroll
				for (int q = 0; q < 4; ++q) tmem_ld_32(ts + (uint32_t)q * 32, v[q]);
#pragma unroll
				for (int q = 0; q < 4; ++q) tmem_ld_wait(v[q]);
				if (__builtin_expect(masked, 0)) { // (edge code out of the loop's straight line: it is 4 KB of instructions)
#pragma unroll
					for (int q = 0; q < 4; ++q) { // bits tested with constants, so that no lane branches
						const uint32_t w = low_bits(top + 1 - q * 32) & (~low_bits(bot - q * 32) | low_bits(sk - q * 32));
#pragma unroll
						for (int c = 0; c < 32; ++c) v[q][c] = (w & (1u << c)) ? v[q][c] : -INFINITY;
					}
				}
				float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
				for (int c = 0; c < 32; c += 2)
#pragma unroll
					for (int q = 0; q < 4; ++q) m4[q] = fmaxf(m4[q], fmaxf(v[q][c], v[q][c + 1]));
				const float mt = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * sl2;
				const bool grow = mt > m + kCtRescaleLog2 || (m == -INFINITY && mt != -INFINITY);
				const float mn = grow ? mt : m;
				if (__builtin_expect(__any_sync(0xFFFFFFFFu, grow && m != -INFINITY), 0)) {
					// S is complete, so every earlier product is: O holds still
					const float f = grow && m != -INFINITY ? ex2_approx(m - mn) : 1.0f;
					l *= f;
#pragma unroll 1
					for (int c = 0; c < HD; c += 16) tmem_scale_16(to + (uint32_t)c, f);
				}
				m = mn;
				const float mu = m == -INFINITY ? 0.0f : m; // nothing seen yet: 2^(-inf) = 0
				const uint64_t mux2 = f2(-mu, -mu);
				// V rows that no row of the item sees become zeros, ahead of P
				if (__builtin_expect(ragged, 0)) {
					ok = wait(kCtFull + vstage, vphase);
					if (!ok) break;
					const int k = k0 + r;
					if (k >= hi || (k < lo && k >= n_sink)) {
						uint4* row = reinterpret_cast<uint4*>(ring_s + (size_t)vstage * kTile + (r >> 3) * kGroup + (r & 7) * 128);
#pragma unroll
						for (int h = 0; h < kHalves; ++h)
#pragma unroll
							for (int c = 0; c < 8; ++c) row[h * 64 + ((c + lane) & 7)] = make_uint4(0, 0, 0, 0); // eight lanes, eight bank groups
					}
					asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
				}
#pragma unroll
				for (int q = 0; q < 4; ++q) {
					uint32_t pk[16];
#pragma unroll
					for (int c = 0; c < 16; ++c) {
						const uint64_t x = f2_fma(f2(v[q][2 * c], v[q][2 * c + 1]), sl2x2, mux2);
						float p0, p1;
						f2_split(x, p0, p1);
						v[q][2 * c] = p0 = ex2_approx(p0);
						v[q][2 * c + 1] = p1 = ex2_approx(p1);
						pk[c] = pack_bf16(p0, p1);
					}
					tmem_st_16regs(ts + (uint32_t)q * 16, pk);
				}
				asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
				tc_fence_before();
				__syncwarp();
				if (lane == 0) mbar_arrive(&bars[kCtP + sub]);
				// the row's sum, while the products run
				uint64_t sum[4] = {0, 0, 0, 0};
#pragma unroll
				for (int c = 0; c < 32; c += 2)
#pragma unroll
					for (int q = 0; q < 4; ++q) sum[q] = f2_add(sum[q], f2(v[q][c], v[q][c + 1]));
				float s0, s1;
				f2_split(f2_add(f2_add(sum[0], sum[1]), f2_add(sum[2], sum[3])), s0, s1);
				l += s0 + s1;
			}
			if (!ok) break;
			// where O goes, and the next item, found while the last product runs
			const bool whole = run.whole();
			uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<bf16*>(a.out) + (uint64_t)(run.q.row0 + tok) * a.out_stride +
			                                      (uint64_t)head * HD);
			// a share of a divided item: [hd / 4][R] float4, so that a warp's stores are whole lines
			float* part = a.part + (size_t)run.slot(worker) * ac_part_floats(a.R, HD);
			const int pr = sub * half_rows + r;
			const float inv = l > 0.0f ? 1.0f / l : 0.0f;
			run.next(a, pre);
			ok = wait(kCtO + sub, o_par);
			if (!ok) break;
			o_par ^= 1u;
			tc_fence_after();
#pragma unroll 1
			for (int c = 0; c < HD; c += 64) {
				float o[2][32];
				tmem_ld_32(to + (uint32_t)c, o[0]);
				tmem_ld_32(to + (uint32_t)c + 32, o[1]);
				tmem_ld_wait(o[0]);
				tmem_ld_wait(o[1]);
				if (r >= valid) {
				} else if (whole) {
#pragma unroll
					for (int u = 0; u < 8; ++u) {
						const float* x = &o[u >> 2][(u & 3) * 8];
						dst[c / 8 + u] = make_uint4(pack_bf16(x[0] * inv, x[1] * inv), pack_bf16(x[2] * inv, x[3] * inv),
						                            pack_bf16(x[4] * inv, x[5] * inv), pack_bf16(x[6] * inv, x[7] * inv));
					}
				} else {
#pragma unroll
					for (int u = 0; u < 16; ++u) {
						const float* x = &o[u >> 3][(u & 7) * 4];
						reinterpret_cast<float4*>(part)[(size_t)(c / 4 + u) * a.R + pr] = make_float4(x[0], x[1], x[2], x[3]);
					}
				}
				__syncwarp(); // together again for the next tcgen05.ld
			}
			if (!whole && r < valid) {
				part[(size_t)a.R * HD + pr] = m;
				part[(size_t)a.R * HD + a.R + pr] = l;
			}
			tc_fence_before(); // the next item's first product overwrites O behind this warpgroup's next P
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
