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

// VP: unit pairs per lane (1, or 2 for rows of more than 32 unit pairs).  Three CTAs an SM: 47 us for 8199 rows of
// 48 x 128 bf16 (4.4 TB/s), against 52 with two CTAs and 128 registers and 49 with four and spills.
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
	const int slot = a.tok_slot[token], pos = a.tok_pos[token];
	if (slot < 0) return; // padding
	const int page_i = pos / a.blk;
	if (slot >= a.n_slots || pos < 0 || pos >= a.n_pos || page_i >= a.pages_per_seq) {
		if (lane == 0) report_err(a.status, kDevKvRange);
		return;
	}
	const int heads = a.H + 2 * a.KV;
	const int h0 = (int)(w % (uint32_t)a.chunks) * a.chunk, h1 = min(heads, h0 + a.chunk);
	const bool writes = h1 > a.H;
	const int page = writes ? a.table[(size_t)slot * a.pages_per_seq + page_i] : 0;
	const bool page_ok = page >= 0 && page < a.n_pages;
	if (writes && !page_ok && lane == 0) report_err(a.status, kDevKvRange);
	const int half_units = a.hd / V / 2, half = a.hd / 2;
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
		if (from >= to) continue;
		// with g = offset + gain: out_i = inv (x_i g_i cos_i - x_(i+h) g_(i+h) sin_i), the other half alike
		float ac[VP][V], bs[VP][V], bc[VP][V], as[VP][V];
		const T* gain = reinterpret_cast<const T*>(kind == 0 ? a.q_gain : a.k_gain);
#pragma unroll
		for (int p = 0; p < VP; ++p) {
			const int u = gl + p * a.lanes;
			float g0[V], g1[V];
#pragma unroll
			for (int i = 0; i < V; ++i) g0[i] = g1[i] = 1.0f;
			if (kind < 2 && gain && mine[p]) {
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
				if (kind < 2 && mine[p]) {
					c = *reinterpret_cast<const float4*>(a.rope_cos + (size_t)pos * half + u * V + i);
					s = *reinterpret_cast<const float4*>(a.rope_sin + (size_t)pos * half + u * V + i);
				}
				const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
				for (int k = 0; k < 4; ++k) {
					ac[p][i + k] = g0[i + k] * cc[k];
					bs[p][i + k] = g1[i + k] * ss[k];
					bc[p][i + k] = g1[i + k] * cc[k];
					as[p][i + k] = g0[i + k] * ss[k];
				}
			}
		}
		uint8_t* dst = kind == 0 ? a.q_out + token * a.q_out_stride + (size_t)(from + grp) * head_bytes
		                         : (kind == 1 ? a.kpool : a.vpool) + slab + (uint64_t)(from + grp - a.H - (kind == 2 ? a.KV : 0)) * a.blk * head_bytes;
		const uint64_t dst_step = (uint64_t)groups * (kind == 0 ? head_bytes : (uint32_t)a.blk * head_bytes);
		const bool stores = kind == 0 || page_ok;
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
				if (kind < 2) {
					float x[VP][V], y[VP][V];
					float ss = 0.0f;
#pragma unroll
					for (int p = 0; p < VP; ++p) {
						unpack_unit(lo[b][p], x[p], (const T*)nullptr);
						unpack_unit(hi[b][p], y[p], (const T*)nullptr);
#pragma unroll
						for (int i = 0; i < V; ++i) ss = fmaf(x[p][i], x[p][i], fmaf(y[p][i], y[p][i], ss));
					}
					float inv = 1.0f;
					if (gain) { // the warp's
						for (int o = a.lanes >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
						inv = rsqrtf(fmaf(ss, a.inv_hd, a.eps));
					}
#pragma unroll
					for (int p = 0; p < VP; ++p) {
						float r0[V], r1[V];
#pragma unroll
						for (int i = 0; i < V; ++i) {
							r0[i] = inv * fmaf(x[p][i], ac[p][i], -(y[p][i] * bs[p][i]));
							r1[i] = inv * fmaf(y[p][i], bc[p][i], x[p][i] * as[p][i]);
						}
						lo[b][p] = pack_unit(r0, (T*)nullptr);
						hi[b][p] = pack_unit(r1, (T*)nullptr);
					}
				}
				if (hb + grp + b * groups < to && stores) {
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
