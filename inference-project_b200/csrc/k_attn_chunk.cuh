// Attention of a ragged batch of new tokens over the paged cache: what its kernels share (the work
// items, their division among workers, the joining of split rows) and the fp32 kernel that serves
// every type and head size.
//
// An item is (sequence, KV head, row tile): the rows of a sequence and KV head are its new tokens times
// the G query heads of the group, row r = token * G + head, R of them to an item, so K and V are read
// once per tile for the whole group.  The keys an item sees come in key tiles of KT positions: those of
// the sinks, then those from the window's start to the last row's position; their number, and what an
// item costs beside them, is its cost.  All costs laid end to end (sequence, head, tile) are cut into
// equal runs, one per worker: a worker may begin inside one item and end inside another, and every worker
// has the same work whatever the lengths are.  Where a cut falls inside an item each worker stores its share
// (O, max, sum), and k_attn_chunk_combine joins them in the workers' order, so a result does not depend
// on which worker finishes first.  Every warp finds its run from the lengths on the device: the host
// needs none of them, and a captured launch follows new lengths.
#pragma once

#include "common.cuh"

namespace inf {

constexpr int kAcMaxSeqs = 4096;

// n / d for 0 <= n < 2^31 by a multiplication: with s = ceil(log2 d) and mul = floor(2^(31+s) / d) + 1 the error
// of n * mul / 2^(31+s) stays below 1 / d (Granlund and Montgomery, PLDI 1994)
struct AcDiv {
	int d;
	uint32_t mul;
	int shift;
	__device__ __forceinline__ int div(int n) const { return (int)(((uint64_t)(uint32_t)n * mul) >> shift); }
	__device__ __forceinline__ int mod(int n) const { return n - div(n) * d; }
};
inline AcDiv ac_div(int d)
{
	int s = 0;
	while ((1ll << s) < d) ++s;
	return {d, (uint32_t)((1ull << (31 + s)) / (uint64_t)d + 1), 31 + s};
}

struct AttnChunkArgs {
	const void* q;
	void* out;
	uint64_t q_stride, out_stride; // elements
	const void* kpool;             // this layer's pages
	const void* vpool;
	const int* table;
	const int* q_start;
	const int* ctx_len;
	const int* seq_slot;           // null: sequence s is slot s
	int n_seqs, n_tokens, max_new;
	int H, KV, G, hd, blk;
	AcDiv group;                   // by G
	int n_slots, pages_per_seq, n_pages;
	int window, n_sink;            // window 0: none
	float scale;
	int* status;
	// division of the work: sequences with more than rows_min and at most rows_max rows per KV head
	// belong to this launch
	int rows_min, rows_max;
	int R;                         // rows of an item
	int workers;
	int min_run;                   // cost of a worker's run at least
	int item_cost;                 // what an item costs beside its key tiles, in key tiles
	float* part;                   // [2 * workers][hd + 2][R] partial O (unnormalised), max (log2 units), sum
	int* jobs;                     // [workers][kAcJobInts]: the item that a worker begins and others end
};

// One job: row0 and rows in q, first head, last worker of the item (0 rows: none).
enum AcJob : int { kAcJobSeq = 0, kAcJobHead = 1, kAcJobRow = 2, kAcJobRows = 3, kAcJobLast = 4, kAcJobInts = 8 };

struct AcSeq {
	int row0, n, ctx, slot; // first row of q, rows, positions, slot
};

// Sequence s, with its numbers checked; n = 0 if it is empty, refused or not of this launch.
__device__ __forceinline__ AcSeq ac_seq(const AttnChunkArgs& a, int s, bool report)
{
	AcSeq q;
	const int b = a.q_start[s], e = a.q_start[s + 1];
	q.row0 = b;
	q.n = 0;
	q.ctx = a.ctx_len[s];
	q.slot = a.seq_slot ? a.seq_slot[s] : s;
	if (e == b) return q;
	int bad = 0;
	if (b < 0 || e < b || e > a.n_tokens || e - b > a.max_new) bad = kDevBadIndex;
	else if (q.slot < 0 || q.slot >= a.n_slots || q.ctx < 0 || q.ctx > a.pages_per_seq * a.blk) bad = kDevKvRange;
	if (bad) {
		if (report) report_err(a.status, bad);
		return q;
	}
	const int64_t rows = (int64_t)(e - b) * a.G;
	if (rows > a.rows_min && rows <= a.rows_max) q.n = e - b;
	return q;
}

// The key tiles of rows [r0, r1) of a sequence: [0, sink) and [first, end); cost >= 1 so that a tile that
// sees nothing is visited (its rows are zeros).
struct AcTiles {
	int lo;    // first position that the window of the tile's first row reaches
	int hi;    // one past the last row's position (<= 0: none)
	int sink, first, end, cost;
};

template <int KT>
__device__ __forceinline__ AcTiles ac_tiles(const AttnChunkArgs& a, const AcSeq& q, int r0, int r1)
{
	AcTiles t;
	const int p0 = q.ctx - q.n + a.group.div(r0), p1 = q.ctx - q.n + a.group.div(r1 - 1);
	t.hi = p1 + 1;
	t.lo = a.window ? max(0, p0 - a.window + 1) : 0;
	const int sinks = min(min(a.n_sink, t.lo), max(t.hi, 0)); // sinks below the window
	t.end = t.hi > 0 ? (t.hi + KT - 1) / KT : 0;
	t.first = min(t.lo / KT, t.end);
	t.sink = min((sinks + KT - 1) / KT, t.first);
	t.cost = max(1, t.sink + t.end - t.first);
	return t;
}
// key tile i (0 .. cost - 1) of an item
__device__ __forceinline__ int ac_tile_at(const AcTiles& t, int i) { return i < t.sink ? i : t.first + i - t.sink; }

// Whether a row at position p sees key k (<= the context).
__device__ __forceinline__ bool ac_sees(const AttnChunkArgs& a, int p, int k)
{
	return k <= p && (a.window == 0 || k > p - a.window || k < a.n_sink);
}

template <int KT>
__device__ __forceinline__ int ac_tile_cost(const AttnChunkArgs& a, const AcSeq& q, int tile)
{
	return ac_tiles<KT>(a, q, tile * a.R, min((tile + 1) * a.R, q.n * a.G)).cost + a.item_cost;
}

// pre[s] = cost of the sequences before s over all heads, pre[n_seqs] = the total.  Every thread of the
// CTA calls it (blockDim a multiple of 32, at most 1024); ends with a barrier.
template <int KT>
__device__ __forceinline__ void ac_prefix(const AttnChunkArgs& a, uint32_t* pre)
{
	const int R = a.R;
	const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
	const bool report = blockIdx.x == 0;
	// a lane per sequence when tiles are few; a warp per sequence, its lanes over the tiles, otherwise
	if (a.max_new * (int64_t)a.G <= 4 * R) {
		for (int s = threadIdx.x; s < a.n_seqs; s += blockDim.x) {
			const AcSeq q = ac_seq(a, s, report);
			uint32_t c = 0;
			for (int t = 0; t * R < q.n * a.G; ++t) c += ac_tile_cost<KT>(a, q, t);
			pre[s + 1] = c * (uint32_t)a.KV;
		}
	} else {
		for (int s = warp; s < a.n_seqs; s += warps) {
			const AcSeq q = ac_seq(a, s, report && lane == 0);
			const int rows = q.n * a.G;
			uint32_t c = 0;
			for (int t = lane; t * R < rows; t += kWarp) c += ac_tile_cost<KT>(a, q, t);
#pragma unroll
			for (int o = 16; o > 0; o >>= 1) c += __shfl_xor_sync(0xFFFFFFFFu, c, o);
			if (lane == 0) pre[s + 1] = c * (uint32_t)a.KV;
		}
	}
	if (threadIdx.x == 0) pre[0] = 0;
	__syncthreads();
	if (warp == 0) {
		// in 64 bits: sequences that name the same rows over and over (q_start going back and forth) cost more than
		// the tokens allow, and such a call does nothing
		uint64_t carry = 0;
		for (int base = 0; base < a.n_seqs; base += kWarp) {
			const int s = base + lane;
			uint64_t v = s < a.n_seqs ? pre[s + 1] : 0u;
#pragma unroll
			for (int o = 1; o < 32; o <<= 1) {
				const uint64_t y = __shfl_up_sync(0xFFFFFFFFu, v, o);
				if (lane >= o) v += y;
			}
			if (s < a.n_seqs) pre[s + 1] = (uint32_t)(carry + v);
			carry += __shfl_sync(0xFFFFFFFFu, v, 31);
		}
		if (carry > 0x7FFFFFFFull) {
			__syncwarp();
			for (int s = lane; s < a.n_seqs; s += kWarp) pre[s + 1] = 0;
			if (report && lane == 0) report_err(a.status, kDevBadIndex);
		}
	}
	__syncthreads();
}

// A worker's run of the laid-out costs, walked item by item (every lane of the warp holds the same).  Lengths are
// read again at every sequence; where they are no longer those of the prefix (a caller that changed them under
// the kernel) the run ends, or goes on over positions inside the tables.
// kOneTile: sequences of at most R rows only.
template <int KT, bool kOneTile = false>
struct AcRun {
	uint32_t at, end, run; // position and end of the run, length of every run
	int s, h, tile, tiles;
	AcSeq q;
	AcTiles t;
	uint32_t item;         // where the current item begins

	__device__ __forceinline__ bool done() const { return at >= end; }
	// this worker's key tiles of the item: [from, to), never none.  The item's own cost lies ahead of its tiles; a run
	// that ends within it leaves the item to the next worker.
	__device__ __forceinline__ int from() const { return max(0, (int)(at - item) - own_); }
	__device__ __forceinline__ int to() const { return min((int)(end - item) - own_, t.cost); }
	__device__ __forceinline__ bool whole() const { return from() == 0 && to() == t.cost; }
	__device__ __forceinline__ int rows() const { return min(r_, rows_ - tile * r_); }
	// slot of the partial: a worker ends at most one item that began before it and begins at most one
	// that ends after it
	__device__ __forceinline__ int slot(int worker) const { return 2 * worker + (from() == 0 ? 1 : 0); }
	__device__ __forceinline__ int last_worker() const { return (int)((item + (uint32_t)(own_ + t.cost) - 1) / run); }
	int r_, rows_, own_; // rows of an item, rows of the sequence, the items' own cost

	__device__ __forceinline__ void tile_of(const AttnChunkArgs& a)
	{
		t = ac_tiles<KT>(a, q, tile * r_, min((tile + 1) * r_, rows_));
		if ((int)(end - item) <= own_) at = end;
	}

	__device__ __forceinline__ void sequence(const AttnChunkArgs& a)
	{
		q = ac_seq(a, s, false);
		rows_ = q.n * a.G;
		tiles = (rows_ + r_ - 1) / r_;
		if (rows_ == 0) at = end; // lengths that changed
	}

	// by a whole warp
	__device__ __forceinline__ void begin(const AttnChunkArgs& a, const uint32_t* pre, int worker)
	{
		const int lane = threadIdx.x & 31;
		const uint32_t total = pre[a.n_seqs];
		run = max((uint32_t)a.min_run, (total + (uint32_t)a.workers - 1) / (uint32_t)a.workers);
		const uint64_t b = (uint64_t)run * (uint32_t)worker;
		at = b < total ? (uint32_t)b : total;
		end = (uint32_t)min(b + run, (uint64_t)total);
		r_ = a.R;
		own_ = a.item_cost;
		if (done()) return;
		int l = 0, r = a.n_seqs; // the last s with pre[s] <= at
		while (r - l > 1) {
			const int m = (l + r) >> 1;
			if (pre[m] <= at) l = m;
			else r = m;
		}
		s = l;
		sequence(a);
		if (done()) return;
		const uint32_t per_head = (pre[s + 1] - pre[s]) / (uint32_t)a.KV;
		const uint32_t in = at - pre[s];
		h = (int)(in / per_head);
		uint32_t left = in % per_head;
		item = at - left;
		if (kOneTile) {
			tile = 0;
			tile_of(a);
			if (from() >= t.cost) at = end; // lengths that changed
			return;
		}
		// the tile that holds `left`: 32 tiles at a time
		bool found = false;
		for (tile = 0; tile < tiles && !found; tile += found ? 0 : kWarp) {
			const int my = tile + lane;
			const uint32_t c = my < tiles ? (uint32_t)ac_tile_cost<KT>(a, q, my) : 0u;
			uint32_t x = c;
#pragma unroll
			for (int o = 1; o < 32; o <<= 1) {
				const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, x, o);
				if (lane >= o) x += y;
			}
			const unsigned hit = __ballot_sync(0xFFFFFFFFu, x > left);
			const uint32_t all = __shfl_sync(0xFFFFFFFFu, x, 31);
			if (hit) {
				const int k = __ffs(hit) - 1;
				item += __shfl_sync(0xFFFFFFFFu, x - c, k);
				tile += k;
				found = true;
			} else {
				left -= all;
				item += all;
			}
		}
		if (found) tile_of(a);
		else at = end; // lengths that changed
	}

	__device__ __forceinline__ void next(const AttnChunkArgs& a, const uint32_t* pre)
	{
		item += (uint32_t)(t.cost + own_);
		at = item;
		if (done()) return;
		if (++tile == tiles) {
			tile = 0;
			if (++h == a.KV) {
				h = 0;
				do ++s;
				while (s < a.n_seqs && pre[s + 1] == pre[s]);
				if (s >= a.n_seqs) { // lengths that changed
					at = end;
					return;
				}
				sequence(a);
				if (done()) return;
			}
		}
		tile_of(a);
	}
};

// The record of an item that worker `w` begins and does not end (one lane calls it), or of none.
__device__ __forceinline__ void ac_job(const AttnChunkArgs& a, int w) { a.jobs[(size_t)w * kAcJobInts + kAcJobRows] = 0; }
template <typename Run>
__device__ __forceinline__ void ac_job(const AttnChunkArgs& a, int w, const Run& run)
{
	int* j = a.jobs + (size_t)w * kAcJobInts;
	j[kAcJobSeq] = run.q.row0;
	j[kAcJobHead] = run.h;
	j[kAcJobRow] = run.tile * a.R;
	j[kAcJobRows] = run.rows();
	j[kAcJobLast] = min(run.last_worker(), a.workers - 1); // (lengths that changed)
}

// floats of one partial: R rows of O, each row's max and sum
__host__ __device__ constexpr size_t ac_part_floats(int R, int hd) { return (size_t)R * (hd + 2); }

// Joins the shares of every item that a cut divides: blockIdx.x is the worker that began it, blockIdx.y a
// block of 32 rows.  A partial holds O as [hd / 4][R] float4, then the rows' max and sum.
//   m = max_i m_i,  O = sum_i 2^(m_i - m) O_i,  l = sum_i 2^(m_i - m) l_i,  out = O / l
// A lane owns a row and, where the item has fewer than 32, every 32 / rows-th share (reads of a row block are
// whole lines, and a long context's many shares are read side by side); the warps share the head dims.
constexpr int kAcCombineThreads = 256;
template <typename T>
__global__ void __launch_bounds__(kAcCombineThreads) k_attn_chunk_combine(const AttnChunkArgs a)
{
	const int R = a.R;
	pdl_wait();
	pdl_trigger();
	const int w0 = blockIdx.x;
	const int* j = a.jobs + (size_t)w0 * kAcJobInts;
	const int rows = j[kAcJobRows] - (int)blockIdx.y * 32; // of this block
	if (rows <= 0) return;
	int wide = 1; // lanes of a row block: a power of two
	while (wide < min(rows, kWarp)) wide <<= 1;
	const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, step = kWarp / wide;
	const bool on = (lane & (wide - 1)) < rows;
	const int r = (int)blockIdx.y * 32 + (on ? lane & (wide - 1) : 0), first = w0 + lane / wide;
	const int last = j[kAcJobLast], hd4 = a.hd / 4;
	const size_t pf = ac_part_floats(R, a.hd);
	// the beginner's share is its second slot, the others' their first
	auto part = [&](int w) { return a.part + (size_t)(2 * w + (w == w0 ? 1 : 0)) * pf; };
	float m = -INFINITY;
#pragma unroll 4
	for (int w = first; w <= last; w += step) m = fmaxf(m, part(w)[(size_t)R * a.hd + r]);
	for (int o = wide; o < kWarp; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
	if (m == -INFINITY) m = 0.0f; // every share without keys: weights of 2^-inf = 0
	const int fr = j[kAcJobRow] + r;
	T* out = reinterpret_cast<T*>(a.out) + (size_t)(j[kAcJobSeq] + a.group.div(fr)) * a.out_stride +
	         (size_t)(j[kAcJobHead] * a.G + a.group.mod(fr)) * a.hd;
	constexpr int kWarps = kAcCombineThreads / kWarp, kCols = 4;
	for (int c0 = warp * kCols; c0 < hd4; c0 += kWarps * kCols) {
		float4 o[kCols];
		float l = 0.0f;
#pragma unroll
		for (int c = 0; c < kCols; ++c) o[c] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
		for (int w = first; w <= last; w += step) {
			const float* p = part(w);
			const float f = exp2f(p[(size_t)R * a.hd + r] - m);
			l = fmaf(f, p[(size_t)R * a.hd + R + r], l);
#pragma unroll
			for (int c = 0; c < kCols; ++c) {
				if (c0 + c >= hd4) continue;
				const float4 v = reinterpret_cast<const float4*>(p)[(size_t)(c0 + c) * R + r];
				o[c].x = fmaf(f, v.x, o[c].x);
				o[c].y = fmaf(f, v.y, o[c].y);
				o[c].z = fmaf(f, v.z, o[c].z);
				o[c].w = fmaf(f, v.w, o[c].w);
			}
		}
		for (int s = wide; s < kWarp; s <<= 1) {
			l += __shfl_xor_sync(0xFFFFFFFFu, l, s);
#pragma unroll
			for (int c = 0; c < kCols; ++c) {
				o[c].x += __shfl_xor_sync(0xFFFFFFFFu, o[c].x, s);
				o[c].y += __shfl_xor_sync(0xFFFFFFFFu, o[c].y, s);
				o[c].z += __shfl_xor_sync(0xFFFFFFFFu, o[c].z, s);
				o[c].w += __shfl_xor_sync(0xFFFFFFFFu, o[c].w, s);
			}
		}
		if (!on || lane >= wide) continue;
		const float inv = l > 0.0f ? 1.0f / l : 0.0f;
		// a row's 16 dims as 16-byte stores (single values, each lane in another row, had taken 50 us for 39 MB
		// of shares); head_dim is a multiple of 16 bytes, so a last short block is whole units too
#pragma unroll
		for (int u = 0; u < (int)(kCols * 4 * sizeof(T) / 16); ++u) {
			constexpr int kPer = 16 / sizeof(T) / 4; // float4 per unit
			if (c0 + u * kPer >= hd4) continue;
			float x[16 / sizeof(T)];
#pragma unroll
			for (int c = 0; c < kPer; ++c) {
				const float4& v = o[u * kPer + c];
				x[4 * c] = v.x * inv;
				x[4 * c + 1] = v.y * inv;
				x[4 * c + 2] = v.z * inv;
				x[4 * c + 3] = v.w * inv;
			}
			*reinterpret_cast<uint4*>(out + 4 * (c0 + u * kPer)) = pack_unit(x, (T*)nullptr);
		}
	}
}

// ---- the fp32 kernel ------------------------------------------------------------------
// Every type, head size, group and page size; a CTA of four warps is a worker.  Tiles of 16 rows x 32
// keys: K and V rows go to shared memory as fp32, a lane owns a key for the scores (four rows of its
// warp at a time) and head dims for P.V.  Bound by shared-memory reads: per key and four head dims one
// 16-byte read of K and one of every row's q for 16 FMAs.  It serves the fp32 decoder (head_dim 48) and
// what the tensor-core kernels do not take.
constexpr int kAfR = 16;
constexpr int kAfKT = 32;
constexpr int kAfThreads = 128;
constexpr int kAfRows = kAfR / (kAfThreads / kWarp); // rows per warp

// q [16][hd], K and V [32][hd + 4] each, P [16][32]
__host__ __device__ constexpr size_t attn_chunk_f32_smem(int hd, int n_seqs)
{
	return ((size_t)kAfR * hd + (size_t)2 * kAfKT * (hd + 4) + kAfR * kAfKT) * 4 + (size_t)(n_seqs + 1) * 4;
}

// VPL: groups of 4 head dims per lane (head_dim <= 128 VPL)
template <typename T, int VPL>
__global__ void __launch_bounds__(kAfThreads) k_attn_chunk_f32(const AttnChunkArgs a)
{
	extern __shared__ __align__(16) float af_smem[];
	pdl_wait();
	pdl_trigger();
	const int hd = a.hd, ld = hd + 4, hd4 = hd / 4;
	float* q_s = af_smem;                 // [16][hd], scaled to log2 units
	float* k_s = q_s + kAfR * hd;         // [32][ld]
	float* v_s = k_s + kAfKT * ld;        // [32][ld]
	float* p_s = v_s + kAfKT * ld;        // [16][32]
	uint32_t* pre = reinterpret_cast<uint32_t*>(p_s + kAfR * kAfKT);
	const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, worker = blockIdx.x;
	ac_prefix<kAfKT>(a, pre);
	AcRun<kAfKT> run;
	run.begin(a, pre, worker);
	if (threadIdx.x == 0) ac_job(a, worker);
	const float sl2 = a.scale * 1.4426950408889634f;
	constexpr int V = Store<T>::kVec;
	for (; !run.done(); run.next(a, pre)) {
		const int rows = run.rows(), r0 = run.tile * kAfR;
		const AcTiles t = run.t;
		const int base_pos = run.q.ctx - run.q.n;
		__syncthreads(); // q_s is free
		for (int u = threadIdx.x; u < kAfR * (hd / V); u += kAfThreads) {
			const int r = u / (hd / V), c = u % (hd / V);
			float f[V];
			uint4 v = make_uint4(0, 0, 0, 0);
			if (r < rows) {
				const int fr = r0 + r;
				v = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.q) + (size_t)(run.q.row0 + a.group.div(fr)) * a.q_stride +
				                                   (size_t)(run.h * a.G + a.group.mod(fr)) * hd)[c];
			}
			unpack_unit(v, f, (const T*)nullptr);
#pragma unroll
			for (int i = 0; i < V; ++i) q_s[r * hd + c * V + i] = f[i] * sl2;
		}
		float4 o[kAfRows][VPL];
		float m[kAfRows], l[kAfRows];
		int pos[kAfRows];
#pragma unroll
		for (int i = 0; i < kAfRows; ++i) {
			m[i] = -INFINITY;
			l[i] = 0.0f;
			const int r = warp * kAfRows + i;
			pos[i] = r < rows ? base_pos + a.group.div(r0 + r) : -1;
#pragma unroll
			for (int v = 0; v < VPL; ++v) o[i][v] = make_float4(0.f, 0.f, 0.f, 0.f);
		}
		for (int kt = run.from(); kt < run.to(); ++kt) {
			const int k0 = ac_tile_at(t, kt) * kAfKT;
			// the tile's 32 rows of K and of V; rows that no row of the item sees are zeros, so that nothing they
			// hold reaches a sum
			__syncthreads(); // the tile before it is read
			for (int u = threadIdx.x; u < kAfKT * (hd / V); u += kAfThreads) {
				const int k = k0 + u / (hd / V), c = u % (hd / V);
				uint4 x[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
				if (k < t.hi && (k >= t.lo || k < a.n_sink)) {
					const int page = a.table[(size_t)run.q.slot * a.pages_per_seq + k / a.blk];
					if (page >= 0 && page < a.n_pages) {
						const size_t at = (((size_t)page * a.KV + run.h) * a.blk + k % a.blk) * hd;
						x[0] = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.kpool) + at)[c];
						x[1] = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.vpool) + at)[c];
					} else {
						report_err(a.status, kDevKvRange);
					}
				}
#pragma unroll
				for (int kv = 0; kv < 2; ++kv) {
					float f[V];
					unpack_unit(x[kv], f, (const T*)nullptr);
#pragma unroll
					for (int i = 0; i < V; i += 4)
						*reinterpret_cast<float4*>((kv ? v_s : k_s) + (size_t)(k - k0) * ld + c * V + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
				}
			}
			__syncthreads();
			float sc[kAfRows];
#pragma unroll
			for (int i = 0; i < kAfRows; ++i) sc[i] = 0.0f;
			for (int d = 0; d < hd; d += 4) {
				const float4 kk = *reinterpret_cast<const float4*>(k_s + (size_t)lane * ld + d);
#pragma unroll
				for (int i = 0; i < kAfRows; ++i) {
					const float4 qq = *reinterpret_cast<const float4*>(q_s + (warp * kAfRows + i) * hd + d);
					sc[i] = fmaf(qq.x, kk.x, fmaf(qq.y, kk.y, fmaf(qq.z, kk.z, fmaf(qq.w, kk.w, sc[i]))));
				}
			}
#pragma unroll
			for (int i = 0; i < kAfRows; ++i) {
				const bool sees = pos[i] >= 0 && ac_sees(a, pos[i], k0 + lane);
				const float s = sees ? sc[i] : -INFINITY;
				const float mn = fmaxf(m[i], warp_max(s));
				// no key seen so far (mn -inf): weights and the factor are zero
				const float f = m[i] == -INFINITY ? 0.0f : exp2f(m[i] - mn);
				const float p = sees ? exp2f(s - mn) : 0.0f;
				m[i] = mn;
				l[i] = l[i] * f + warp_sum(p);
				p_s[(warp * kAfRows + i) * kAfKT + lane] = p;
#pragma unroll
				for (int v = 0; v < VPL; ++v) {
					o[i][v].x *= f;
					o[i][v].y *= f;
					o[i][v].z *= f;
					o[i][v].w *= f;
				}
			}
			__syncwarp(); // the warp's own rows of P
			for (int k = 0; k < kAfKT; k += 4) {
				float4 p[kAfRows];
#pragma unroll
				for (int i = 0; i < kAfRows; ++i) p[i] = *reinterpret_cast<const float4*>(p_s + (warp * kAfRows + i) * kAfKT + k);
#pragma unroll
				for (int v = 0; v < VPL; ++v) {
					const int c = lane + v * kWarp;
					if (c >= hd4) continue;
#pragma unroll
					for (int kk = 0; kk < 4; ++kk) {
						const float4 x = *reinterpret_cast<const float4*>(v_s + (size_t)(k + kk) * ld + c * 4);
#pragma unroll
						for (int i = 0; i < kAfRows; ++i) {
							const float w = kk == 0 ? p[i].x : kk == 1 ? p[i].y : kk == 2 ? p[i].z : p[i].w;
							o[i][v].x = fmaf(w, x.x, o[i][v].x);
							o[i][v].y = fmaf(w, x.y, o[i][v].y);
							o[i][v].z = fmaf(w, x.z, o[i][v].z);
							o[i][v].w = fmaf(w, x.w, o[i][v].w);
						}
					}
				}
			}
		}
		const bool whole = run.whole();
		float* part = a.part + (size_t)run.slot(worker) * ac_part_floats(kAfR, hd);
#pragma unroll
		for (int i = 0; i < kAfRows; ++i) {
			const int r = warp * kAfRows + i;
			if (r >= rows) continue;
			if (whole) {
				const float inv = l[i] > 0.0f ? 1.0f / l[i] : 0.0f;
				const int fr = r0 + r;
				T* out = reinterpret_cast<T*>(a.out) + (size_t)(run.q.row0 + a.group.div(fr)) * a.out_stride + (size_t)(run.h * a.G + a.group.mod(fr)) * hd;
#pragma unroll
				for (int v = 0; v < VPL; ++v) {
					const int c = lane + v * kWarp;
					if (c >= hd4) continue;
					Store<T>::put(out + 4 * c, o[i][v].x * inv);
					Store<T>::put(out + 4 * c + 1, o[i][v].y * inv);
					Store<T>::put(out + 4 * c + 2, o[i][v].z * inv);
					Store<T>::put(out + 4 * c + 3, o[i][v].w * inv);
				}
			} else {
#pragma unroll
				for (int v = 0; v < VPL; ++v) {
					const int c = lane + v * kWarp;
					if (c < hd4) reinterpret_cast<float4*>(part)[(size_t)c * kAfR + r] = o[i][v];
				}
				if (lane == 0) {
					part[(size_t)kAfR * hd + r] = m[i];
					part[(size_t)kAfR * hd + kAfR + r] = l[i];
				}
			}
		}
		if (!whole && run.from() == 0 && threadIdx.x == 0) ac_job(a, worker, run);
	}
}

} // namespace inf
