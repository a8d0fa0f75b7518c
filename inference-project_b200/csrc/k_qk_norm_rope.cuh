// RMSNorm of every query and key head, rotation by the token's position, and the write of K and V
// into the paged cache, in one pass over the projected rows of new tokens.
//
//   y = x * (1 / sqrt(mean(x^2) + eps)) * (offset + gain)          fp32, one rounding at the end
//   out_i = y_i cos_i - y_(i+h) sin_i,  out_(i+h) = y_(i+h) cos_i + y_i sin_i,   h = head_dim / 2
//
// Bound by HBM: every element is read once and written once.  A group of lanes owns a head, a lane the
// 16-byte units u and u + units/2 of it, so both partners of a rotation are in one lane and the only
// exchange is the sum of squares (3 shuffles for head_dim 128 in bf16: 8 lanes x 2 units).  A warp goes
// through the heads of one token, its groups side by side, and keeps the products of gain, cos and sin in
// registers: per element that leaves the unpacking, the square, one multiply-add and the scale, which the
// SMs issue in about half of the time that HBM takes.
#pragma once

#include "common.cuh"

namespace inf {

constexpr int kQnThreads = 256;
constexpr int kQnBatch = 2; // heads in flight per group

struct QkNormRopeArgs {
	const uint8_t* qkv;
	uint8_t* q_out;
	uint64_t qkv_stride, q_out_stride; // bytes
	const void* q_gain;
	const void* k_gain;
	const float* rope_cos;
	const float* rope_sin;
	const int* tok_slot;
	const int* tok_pos;
	int* status;
	float eps, gain_offset, inv_hd;
	int n_pos;
	uint32_t n_tokens;
	int H, KV, hd, blk;
	uint8_t* kpool; // this layer's
	uint8_t* vpool;
	const int* table;
	int n_slots, pages_per_seq, n_pages;
	int lanes;      // lanes per head, a power of two >= units / 2 / VP
	int chunk;      // heads per warp
	int chunks;     // warps per token
};

// One lane's share of gain, cos and sin.  With g = offset + gain:
//   out_i = inv (x_i g_i cos_i - x_(i+h) g_(i+h) sin_i),  out_(i+h) = inv (x_(i+h) g_(i+h) cos_i + x_i g_i sin_i)
// Two elements to an instruction throughout: the kernel issues for half of the time that it takes.
template <typename T, int VP>
struct QnTurn {
	static constexpr int V = Store<T>::kVec, V2 = V / 2; // elements per unit, pairs of them
	uint64_t ac[VP][V2], nbs[VP][V2], bc[VP][V2], as[VP][V2]; // nbs: negated
	bool norm;

	__device__ __forceinline__ void load(const QkNormRopeArgs& a, const T* gain, int pos, int gl, const bool (&mine)[VP])
	{
		const int half_units = a.hd / V / 2, half = a.hd / 2;
		norm = gain != nullptr;
#pragma unroll
		for (int p = 0; p < VP; ++p) {
			const int u = gl + p * a.lanes;
			float g0[V], g1[V];
#pragma unroll
			for (int i = 0; i < V; ++i) g0[i] = g1[i] = 1.0f;
			if (gain && mine[p]) {
				unpack_unit(reinterpret_cast<const uint4*>(gain)[u], g0, (const T*)nullptr);
				unpack_unit(reinterpret_cast<const uint4*>(gain)[u + half_units], g1, (const T*)nullptr);
#pragma unroll
				for (int i = 0; i < V; ++i) {
					g0[i] += a.gain_offset;
					g1[i] += a.gain_offset;
				}
			}
#pragma unroll
			for (int i = 0; i < V; i += 4) {
				float4 c = make_float4(1.f, 1.f, 1.f, 1.f), s = make_float4(0.f, 0.f, 0.f, 0.f);
				if (mine[p]) {
					c = *reinterpret_cast<const float4*>(a.rope_cos + (size_t)pos * half + u * V + i);
					s = *reinterpret_cast<const float4*>(a.rope_sin + (size_t)pos * half + u * V + i);
				}
				const uint64_t cc[2] = {f2(c.x, c.y), f2(c.z, c.w)}, ss[2] = {f2(s.x, s.y), f2(s.z, s.w)};
#pragma unroll
				for (int k = 0; k < 2; ++k) {
					const int e = i + 2 * k;
					const uint64_t a0 = f2(g0[e], g0[e + 1]), a1 = f2(g1[e], g1[e + 1]);
					ac[p][e / 2] = f2_mul(a0, cc[k]);
					nbs[p][e / 2] = f2_mul(f2(-g1[e], -g1[e + 1]), ss[k]);
					bc[p][e / 2] = f2_mul(a1, cc[k]);
					as[p][e / 2] = f2_mul(a0, ss[k]);
				}
			}
		}
	}

	// one head, its units u and u + units / 2 in lo and hi (zeros in lanes without a share); by the whole warp
	__device__ __forceinline__ void turn(const QkNormRopeArgs& a, uint4 (&lo)[VP], uint4 (&hi)[VP]) const
	{
		uint64_t x[VP][V2], y[VP][V2];
		uint64_t s0 = 0, s1 = 0;
#pragma unroll
		for (int p = 0; p < VP; ++p) {
			float v[V], w[V];
			unpack_unit(lo[p], v, (const T*)nullptr);
			unpack_unit(hi[p], w, (const T*)nullptr);
#pragma unroll
			for (int i = 0; i < V2; ++i) {
				x[p][i] = f2(v[2 * i], v[2 * i + 1]);
				y[p][i] = f2(w[2 * i], w[2 * i + 1]);
				s0 = f2_fma(x[p][i], x[p][i], s0);
				s1 = f2_fma(y[p][i], y[p][i], s1);
			}
		}
		float inv = 1.0f;
		if (norm) {
			float u, v;
			f2_split(f2_add(s0, s1), u, v);
			float ss = u + v;
			for (int o = a.lanes >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
			inv = rsqrtf(fmaf(ss, a.inv_hd, a.eps));
		}
		const uint64_t inv2 = f2(inv, inv);
#pragma unroll
		for (int p = 0; p < VP; ++p) {
			float r0[V], r1[V];
#pragma unroll
			for (int i = 0; i < V2; ++i) {
				f2_split(f2_mul(inv2, f2_fma(x[p][i], ac[p][i], f2_mul(y[p][i], nbs[p][i]))), r0[2 * i], r0[2 * i + 1]);
				f2_split(f2_mul(inv2, f2_fma(y[p][i], bc[p][i], f2_mul(x[p][i], as[p][i]))), r1[2 * i], r1[2 * i + 1]);
			}
			lo[p] = pack_unit(r0, (T*)nullptr);
			hi[p] = pack_unit(r1, (T*)nullptr);
		}
	}
};

// The page of a token and whether it is done at all: 0 skipped, 1 queries only (its page is missing), 2 all.
__device__ __forceinline__ int qn_token(const QkNormRopeArgs& a, int slot, int pos, bool writes, int* page)
{
	if (slot < 0) return 0; // padding
	const bool first = (threadIdx.x & 31) == 0;
	const int page_i = pos / a.blk;
	if (slot >= a.n_slots || pos < 0 || pos >= a.n_pos || page_i >= a.pages_per_seq) {
		if (first) report_err(a.status, kDevKvRange);
		return 0;
	}
	*page = 0;
	if (!writes) return 2;
	*page = a.table[(size_t)slot * a.pages_per_seq + page_i];
	if (*page >= 0 && *page < a.n_pages) return 2;
	if (first) report_err(a.status, kDevKvRange);
	return 1;
}

// VP: unit pairs per lane (1, or 2 for rows of more than 32 unit pairs).  Three CTAs an SM: 44 us for 8199 rows of
// 48 x 128 bf16 (4.6 TB/s); two CTAs with more registers and four with spills were 10% and 4% slower.  Filling
// shared-memory rings by bulk copies ahead of the arithmetic measured the same (45 us): the loads' latency is
// covered, what is left is the arithmetic's issue and that a warp slot gets 2.3 tokens on average but 3 at most.
template <typename T, int VP>
__global__ void __launch_bounds__(kQnThreads, VP == 1 ? 3 : 1) k_qk_norm_rope_rows(const QkNormRopeArgs a)
{
	constexpr int V = Store<T>::kVec; // elements per unit
	pdl_wait();
	pdl_trigger();
	const int lane = threadIdx.x & 31, gl = lane & (a.lanes - 1), grp = lane / a.lanes, groups = kWarp / a.lanes;
	const uint64_t w = (uint64_t)blockIdx.x * (kQnThreads / kWarp) + threadIdx.x / kWarp;
	const uint64_t token = w / (uint32_t)a.chunks; // a warp: `chunk` heads of one token
	if (token >= a.n_tokens) return;
	const int heads = a.H + 2 * a.KV;
	const int h0 = (int)(w % (uint32_t)a.chunks) * a.chunk, h1 = min(heads, h0 + a.chunk);
	const int pos = a.tok_pos[token];
	int page = 0;
	const int what = qn_token(a, a.tok_slot[token], pos, h1 > a.H, &page);
	if (what == 0) return;
	const int half_units = a.hd / V / 2;
	const uint8_t* row = a.qkv + token * a.qkv_stride;
	const uint32_t head_bytes = (uint32_t)a.hd * sizeof(T);
	const uint64_t slab = ((uint64_t)page * a.KV * a.blk + pos % a.blk) * head_bytes; // head 0's row of the page
	bool mine[VP];
#pragma unroll
	for (int p = 0; p < VP; ++p) mine[p] = gl + p * a.lanes < half_units;
	// the warp's heads in three kinds: queries, keys, values; its groups take them in turn
#pragma unroll 1
	for (int kind = 0; kind < 3; ++kind) {
		const int from = max(h0, kind == 0 ? 0 : kind == 1 ? a.H : a.H + a.KV);
		const int to = min(h1, kind == 0 ? a.H : kind == 1 ? a.H + a.KV : heads);
		if (from >= to || (kind > 0 && what == 1)) continue;
		QnTurn<T, VP> turn;
		if (kind < 2) turn.load(a, reinterpret_cast<const T*>(kind == 0 ? a.q_gain : a.k_gain), pos, gl, mine);
		uint8_t* dst = kind == 0 ? a.q_out + token * a.q_out_stride + (size_t)(from + grp) * head_bytes
		                         : (kind == 1 ? a.kpool : a.vpool) + slab + (uint64_t)(from + grp - a.H - (kind == 2 ? a.KV : 0)) * a.blk * head_bytes;
		const uint64_t dst_step = (uint64_t)groups * (kind == 0 ? head_bytes : (uint32_t)a.blk * head_bytes);
		for (int hb = from; hb < to; hb += kQnBatch * groups) {
			uint4 lo[kQnBatch][VP], hi[kQnBatch][VP];
#pragma unroll
			for (int b = 0; b < kQnBatch; ++b)
#pragma unroll
				for (int p = 0; p < VP; ++p) {
					lo[b][p] = hi[b][p] = make_uint4(0, 0, 0, 0);
					if (mine[p] && hb + grp + b * groups < to) {
						const uint4* src = reinterpret_cast<const uint4*>(row + (size_t)(hb + grp + b * groups) * head_bytes);
						lo[b][p] = src[gl + p * a.lanes];
						hi[b][p] = src[gl + p * a.lanes + half_units];
					}
				}
#pragma unroll
			for (int b = 0; b < kQnBatch; ++b) {
				if (kind < 2) turn.turn(a, lo[b], hi[b]);
				if (hb + grp + b * groups < to) {
#pragma unroll
					for (int p = 0; p < VP; ++p) {
						if (!mine[p]) continue;
						reinterpret_cast<uint4*>(dst)[gl + p * a.lanes] = lo[b][p];
						reinterpret_cast<uint4*>(dst)[gl + p * a.lanes + half_units] = hi[b][p];
					}
				}
				dst += dst_step;
			}
		}
	}
}

} // namespace inf
