// Copying, freeing, forking and compacting the pages of a paged KV cache.
//
// Bookkeeping is integer work on two device arrays, the block tables and one reference count per
// page; nothing depends on the order in which threads run: pages are handed out by a scan over ids,
// reference counts change by integer adds, a table entry is given up by the one thread that exchanges
// it.  The data movement is a plain copy, bound by HBM (two bytes moved per byte copied): a warp
// owns a contiguous run of 4 KB slices, each lane with eight 16-byte loads in flight before the
// first store.
#pragma once

#include "common.cuh"

namespace inf {

constexpr int kPgThreads = 256;
constexpr int kPgUnroll = 8;                             // 16-byte units per lane and slice
constexpr uint32_t kPgSlice = kPgUnroll * kWarp * 16;    // 4096 bytes
constexpr int kPlanThreads = 1024;
constexpr uint32_t kCompactMaxPages = 1u << 19;          // a bit and a 32nd of a count each in the plan's shared memory: 128 KB

struct PagePools {
	uint8_t* k;
	uint8_t* v;
	uint64_t layer_stride;
	uint32_t n_layers;
	uint32_t page_bytes;  // one page of K (or V) of one layer
	uint32_t head_bytes;  // one head of it
	uint32_t row_bytes;   // one position of one head
	int n_pages;
};

// Segment `seg` of a page: layer seg / 2, K (even) or V (odd).
__device__ __forceinline__ uint8_t* page_segment(const PagePools& P, uint32_t seg, int page)
{
	return ((seg & 1u) ? P.v : P.k) + (uint64_t)(seg >> 1) * P.layer_stride + (uint64_t)page * P.page_bytes;
}

// up to kPgSlice bytes (a multiple of 16), by one warp
__device__ __forceinline__ void warp_copy(uint8_t* dst, const uint8_t* src, uint32_t bytes)
{
	const int lane = threadIdx.x & 31;
	const uint32_t units = bytes >> 4;
	uint4 r[kPgUnroll];
#pragma unroll
	for (int k = 0; k < kPgUnroll; ++k) {
		const uint32_t u = (uint32_t)k * kWarp + lane;
		if (u < units) r[k] = reinterpret_cast<const uint4*>(src)[u];
	}
#pragma unroll
	for (int k = 0; k < kPgUnroll; ++k) {
		const uint32_t u = (uint32_t)k * kWarp + lane;
		if (u < units) reinterpret_cast<uint4*>(dst)[u] = r[k];
	}
}

// The whole-page copies of `n` pairs, spread over every warp of the grid; pair(i, src, dst) gives the
// ids of pair i and whether it is copied (called by the whole warp, i uniform).
template <typename F>
__device__ __forceinline__ void copy_pairs(const PagePools& P, uint32_t n, F pair)
{
	const uint32_t spp = (P.page_bytes + kPgSlice - 1) / kPgSlice; // slices per page and segment
	const uint32_t per_pair = 2 * P.n_layers * spp;
	const uint64_t total = (uint64_t)n * per_pair;
	const uint64_t warps = (uint64_t)gridDim.x * (blockDim.x / kWarp);
	const uint64_t w = (uint64_t)blockIdx.x * (blockDim.x / kWarp) + threadIdx.x / kWarp;
	const uint64_t begin = total * w / warps, end = total * (w + 1) / warps;
	if (begin >= end) return;
	uint32_t i = (uint32_t)(begin / per_pair);
	uint32_t in = (uint32_t)(begin % per_pair);
	uint32_t seg = in / spp, sl = in % spp;
	int src = 0, dst = 0;
	bool ok = pair(i, src, dst);
	for (uint64_t x = begin; x < end; ++x) {
		if (ok) {
			const uint32_t off = sl * kPgSlice;
			warp_copy(page_segment(P, seg, dst) + off, page_segment(P, seg, src) + off, min(kPgSlice, P.page_bytes - off));
		}
		if (++sl == spp) {
			sl = 0;
			if (++seg == 2 * P.n_layers) {
				seg = 0;
				if (++i < n && x + 1 < end) ok = pair(i, src, dst);
			}
		}
	}
}

// ---- copy -----------------------------------------------------------------------------
struct PageCopyArgs {
	PagePools P;
	const int* src;
	const int* dst;
	uint32_t n;
	int* status;
};

__global__ void __launch_bounds__(kPgThreads) k_kv_copy_pages(const PageCopyArgs a)
{
	pdl_wait();
	pdl_trigger();
	const int lane = threadIdx.x & 31;
	copy_pairs(a.P, a.n, [&](uint32_t i, int& src, int& dst) {
		src = a.src[i];
		dst = a.dst[i];
		bool ok = src >= 0 && src < a.P.n_pages && dst >= 0 && dst < a.P.n_pages;
		// a page written twice, or read by another pair while it is written, has no order to go by.
		// The scan reads both lists, 8 n bytes from L2, for every pair that a warp enters: nothing beside the copy of
		// pages of many layers (22 layers of 4 x 16 x 64 bf16: 5.4 TB/s at 4000 pairs, 4.5 at 16000), but more than
		// the copy where one layer's small pages go by the thousand (4000 pairs of 16 KB, K and V: 124 us, 20 at the
		// copy rate; of 64 KB: 169 us, 80).
		for (uint32_t j = lane; j < a.n; j += kWarp) ok = ok && !(j < i && a.dst[j] == dst) && a.src[j] != dst;
		ok = __all_sync(0xFFFFFFFFu, ok);
		if (!ok && lane == 0) report_err(a.status, kDevBadIndex);
		return ok;
	});
}

// ---- free -----------------------------------------------------------------------------
struct PageFreeArgs {
	int* table;
	int* refs;
	int n_slots, pages_per_seq, n_pages;
	const int* slot;
	const int* first;
	const int* last;
	int* status;
};

// grid (entries / kPgThreads, n)
__global__ void __launch_bounds__(kPgThreads) k_kv_free(const PageFreeArgs a, uint32_t n)
{
	pdl_wait();
	pdl_trigger();
	for (uint32_t i = blockIdx.y; i < n; i += gridDim.y) {
		const int slot = a.slot[i], first = a.first ? a.first[i] : 0, last = a.last ? a.last[i] : a.pages_per_seq;
		// both ends within the table: entry indices fit 31 bits with a grid's width to spare (pages_per_seq <= 2^30)
		if (slot < 0 || slot >= a.n_slots || first < 0 || first > a.pages_per_seq || last < 0 || last > a.pages_per_seq) {
			if (blockIdx.x == 0 && threadIdx.x == 0) report_err(a.status, kDevBadIndex);
			continue;
		}
		for (int e = first + (int)(blockIdx.x * blockDim.x + threadIdx.x); e < last; e += (int)(gridDim.x * blockDim.x)) {
			// the exchange gives each entry to one thread, however often the call names it
			const int page = atomicExch(a.table + (size_t)slot * a.pages_per_seq + e, -1);
			if (page == -1) continue;
			if (page < 0 || page >= a.n_pages) {
				report_err(a.status, kDevBadIndex);
			} else if (atomicSub(a.refs + page, 1) <= 0) {
				atomicAdd(a.refs + page, 1); // it had none: left as it was
				report_err(a.status, kDevBadIndex);
			}
		}
	}
}

// ---- fork -----------------------------------------------------------------------------
struct ForkJob {
	int src_slot, dst_slot;
	int full;     // shared pages; -1: the fork is refused
	int rows;     // positions in the last, partial page
	int src_page; // that page and its copy (-1: none)
	int dst_page;
};

struct ForkArgs {
	PagePools P;
	int* table;
	int* refs;
	int n_slots, pages_per_seq, kv_block;
	const int* src;
	const int* dst;
	const int* len;
	uint32_t n;
	ForkJob* jobs; // [n]
	int* fresh;    // [n]
	int* status;
};

// Exclusive prefix sum of v over the CTA (kPlanThreads threads); *total = the sum.  Two barriers.
__device__ __forceinline__ uint32_t plan_scan(uint32_t v, uint32_t* total)
{
	__shared__ uint32_t sums[kPlanThreads / kWarp];
	const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
	uint32_t x = v;
#pragma unroll
	for (int o = 1; o < 32; o <<= 1) {
		const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, x, o);
		if (lane >= o) x += y;
	}
	if (lane == 31) sums[warp] = x;
	__syncthreads();
	uint32_t s = sums[lane];
#pragma unroll
	for (int o = 1; o < 32; o <<= 1) {
		const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, s, o);
		if (lane >= o) s += y;
	}
	*total = __shfl_sync(0xFFFFFFFFu, s, 31);
	const uint32_t before = warp ? __shfl_sync(0xFFFFFFFFu, s, warp - 1) : 0u;
	__syncthreads(); // sums may be reused
	return before + x - v;
}

// One CTA: which forks are valid, and which fresh page each partial page gets.
__global__ void __launch_bounds__(kPlanThreads) k_kv_fork_plan(const ForkArgs a)
{
	pdl_wait();
	pdl_trigger();
	const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
	// one warp per fork: its numbers, the other forks' slots (n^2 / 32 steps in all, in one CTA: 30 us a call at 256
	// forks, 146 at 1024, 1.7 ms at 4096), its destination row
	for (uint32_t i = warp; i < a.n; i += kPlanThreads / kWarp) {
		const int s = a.src[i], d = a.dst[i], len = a.len[i];
		bool ok = s >= 0 && s < a.n_slots && d >= 0 && d < a.n_slots && len >= 0 && len <= a.pages_per_seq * a.kv_block;
		for (uint32_t j = lane; j < a.n; j += kWarp) ok = ok && !(j < i && a.dst[j] == d) && a.src[j] != d;
		ok = __all_sync(0xFFFFFFFFu, ok);
		if (ok) {
			const int* row = a.table + (size_t)d * a.pages_per_seq;
			for (int e = lane; e < a.pages_per_seq; e += kWarp) ok = ok && row[e] == -1;
			ok = __all_sync(0xFFFFFFFFu, ok);
		}
		if (lane == 0) {
			ForkJob jb = {s, d, ok ? len / a.kv_block : -1, ok ? len % a.kv_block : 0, -1, -1};
			if (ok && jb.rows) jb.src_page = a.table[(size_t)s * a.pages_per_seq + jb.full];
			if (!ok || jb.src_page < -1 || jb.src_page >= a.P.n_pages) report_err(a.status, kDevBadIndex);
			if (jb.src_page >= a.P.n_pages || jb.src_page < 0) jb.src_page = -1; // a missing page stays missing
			a.jobs[i] = jb;
		}
	}
	__syncthreads(); // the jobs are read back by other threads (global, same CTA)
	uint32_t need = 0;
	for (uint32_t base = 0; base < a.n; base += kPlanThreads) {
		const uint32_t i = base + tid;
		const uint32_t mine = i < a.n && a.jobs[i].src_page >= 0 ? 1u : 0u;
		uint32_t sum;
		const uint32_t rank = need + plan_scan(mine, &sum);
		if (mine) a.jobs[i].dst_page = (int)rank; // the rank until the free pages are known
		need += sum;
	}
	uint32_t found = 0;
	for (int base = 0; base < a.P.n_pages && found < need; base += kPlanThreads) {
		const int p = base + tid;
		const uint32_t mine = p < a.P.n_pages && a.refs[p] == 0 ? 1u : 0u;
		uint32_t sum;
		const uint32_t rank = found + plan_scan(mine, &sum);
		if (mine && rank < need) a.fresh[rank] = p;
		found += sum;
	}
	__syncthreads();
	for (uint32_t i = tid; i < a.n; i += kPlanThreads) {
		const int rank = a.jobs[i].dst_page;
		if (rank < 0) continue;
		if ((uint32_t)rank < found) {
			a.jobs[i].dst_page = a.fresh[rank];
		} else {
			a.jobs[i].full = -1;
			a.jobs[i].src_page = a.jobs[i].dst_page = -1;
			report_err(a.status, kDevNoPages);
		}
	}
}

// Block tables and references of fork blockIdx.x (the first n CTAs), then the partial pages' rows: a
// warp per (fork, layer, K or V, head).
__global__ void __launch_bounds__(kPgThreads) k_kv_fork(const ForkArgs a)
{
	pdl_wait();
	pdl_trigger();
	if (blockIdx.x < a.n) {
		const ForkJob jb = a.jobs[blockIdx.x];
		if (jb.full < 0) return;
		const int* from = a.table + (size_t)jb.src_slot * a.pages_per_seq;
		int* to = a.table + (size_t)jb.dst_slot * a.pages_per_seq; // all -1 so far
		for (int e = threadIdx.x; e < jb.full; e += blockDim.x) {
			const int page = from[e];
			if (page == -1) continue;
			if (page < 0 || page >= a.P.n_pages) {
				report_err(a.status, kDevBadIndex);
				continue;
			}
			atomicAdd(a.refs + page, 1);
			to[e] = page;
		}
		if (threadIdx.x == 0 && jb.dst_page >= 0) {
			to[jb.full] = jb.dst_page;
			atomicAdd(a.refs + jb.dst_page, 1);
		}
		return;
	}
	const uint32_t heads = a.P.page_bytes / a.P.head_bytes, per_fork = 2 * a.P.n_layers * heads;
	const uint64_t total = (uint64_t)a.n * per_fork;
	const uint64_t step = (uint64_t)(gridDim.x - a.n) * (kPgThreads / kWarp);
	for (uint64_t x = (uint64_t)(blockIdx.x - a.n) * (kPgThreads / kWarp) + threadIdx.x / kWarp; x < total; x += step) {
		const ForkJob jb = a.jobs[x / per_fork];
		if (jb.dst_page < 0) continue;
		const uint32_t r = (uint32_t)(x % per_fork), seg = r / heads;
		const uint64_t head = (uint64_t)(r % heads) * a.P.head_bytes;
		const uint32_t bytes = (uint32_t)jb.rows * a.P.row_bytes;
		for (uint32_t off = 0; off < bytes; off += kPgSlice)
			warp_copy(page_segment(a.P, seg, jb.dst_page) + head + off, page_segment(a.P, seg, jb.src_page) + head + off,
			          min(kPgSlice, bytes - off));
	}
}

// ---- compact --------------------------------------------------------------------------
struct CompactArgs {
	PagePools P;
	int* table;
	int* refs;
	int n_slots, pages_per_seq;
	int* map;      // [n_pages] new id of each old page, -1: free
	int* n_live;
	int* n_moves;  // scratch
	int* from;     // [n_pages] scratch: the i-th page that moves
	int* to;       // [n_pages] scratch: where to
	int* status;
};

// One CTA: a bit per page in shared memory, a prefix sum of its words, the list of moves and the map.
__global__ void __launch_bounds__(kPlanThreads) k_kv_compact_plan(const CompactArgs a)
{
	extern __shared__ uint32_t live_s[]; // [words] bits, then [words] pages in use below the word
	pdl_wait();
	pdl_trigger();
	const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
	const int n = a.P.n_pages, words = (n + 31) / 32;
	uint32_t* below = live_s + words;
	for (int w = warp; w < words; w += kPlanThreads / kWarp) {
		const int p = w * 32 + lane;
		const int refs = p < n ? a.refs[p] : 0;
		if (refs < 0) report_err(a.status, kDevBadIndex);
		const uint32_t bits = __ballot_sync(0xFFFFFFFFu, refs > 0);
		if (lane == 0) live_s[w] = bits;
	}
	__syncthreads();
	uint32_t total = 0;
	for (int base = 0; base < words; base += kPlanThreads) {
		const int w = base + tid;
		uint32_t sum;
		const uint32_t x = total + plan_scan(w < words ? __popc(live_s[w]) : 0u, &sum);
		if (w < words) below[w] = x;
		total += sum;
	}
	__syncthreads();
	const int L = (int)total;
	const int lw = L >> 5; // pages in use below id L (L == n: all of them)
	const uint32_t low = L < n ? below[lw] + __popc(live_s[lw] & ((1u << (L & 31)) - 1u)) : total;
	for (int p = tid; p < n; p += kPlanThreads) {
		const uint32_t bits = live_s[p >> 5];
		const uint32_t rank = below[p >> 5] + __popc(bits & ((1u << (p & 31)) - 1u)); // pages in use below p
		const bool live = (bits >> (p & 31)) & 1u;
		if (live && p >= L) a.from[rank - low] = p;
		if (!live && p < L) a.to[p - (int)rank] = p;
	}
	__syncthreads(); // the lists are read back by other threads (global, same CTA)
	for (int p = tid; p < n; p += kPlanThreads) {
		const uint32_t bits = live_s[p >> 5];
		const uint32_t rank = below[p >> 5] + __popc(bits & ((1u << (p & 31)) - 1u));
		const bool live = (bits >> (p & 31)) & 1u;
		a.map[p] = !live ? -1 : p < L ? p : a.to[rank - low];
	}
	if (tid == 0) {
		*a.n_live = L;
		*a.n_moves = (int)(total - low);
	}
}

__global__ void __launch_bounds__(kPgThreads) k_kv_compact(const CompactArgs a)
{
	pdl_wait();
	pdl_trigger();
	const uint32_t moves = (uint32_t)*a.n_moves;
	const uint64_t t = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x, step = (uint64_t)gridDim.x * blockDim.x;
	for (uint64_t i = t; i < moves; i += step) { // the pages moved to are free: no two threads meet
		a.refs[a.to[i]] = a.refs[a.from[i]];
		a.refs[a.from[i]] = 0;
	}
	const uint64_t entries = (uint64_t)a.n_slots * a.pages_per_seq;
	for (uint64_t e = t; e < entries; e += step) {
		const int page = a.table[e];
		if (page == -1) continue;
		const int now = page >= 0 && page < a.P.n_pages ? a.map[page] : -1;
		if (now < 0) report_err(a.status, kDevBadIndex); // no such page, or one without references
		else if (now != page) a.table[e] = now;
	}
	copy_pairs(a.P, moves, [&](uint32_t i, int& src, int& dst) {
		src = a.from[i];
		dst = a.to[i];
		return true;
	});
}

} // namespace inf
