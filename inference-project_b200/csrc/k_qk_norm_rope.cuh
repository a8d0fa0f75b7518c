// RMSNorm of every query and key head, rotation by the token's position, and the write of K and V
// into the paged cache, in one pass over the projected rows of new tokens.
//
//   y = x * (1 / sqrt(mean(x^2) + eps)) * (offset + gain)          fp32, one rounding at the end
//   out_i = y_i cos_i - y_(i+h) sin_i,  out_(i+h) = y_(i+h) cos_i + y_i sin_i,   h = head_dim / 2
//
// Bound by HBM: every element is read once and written once.  A group of lanes owns a head, a lane the
// 16-byte units u and u + units/2 of it, so both partners of a rotation are in one lane and the only
// exchange is the sum of squares (3 shuffles for head_dim 128 in bf16: 8 lanes x 2 units).  A group goes
// through several heads of its token, four at a time with their loads in flight together, and keeps
// the token's cos and sin, which are as many bytes as two bf16 heads, in registers.
#pragma once

#include "common.cuh"

namespace inf {

constexpr int kQnThreads = 256;
constexpr int kQnBatch = 4; // heads in flight per group

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
	float eps, gain_offset;
	int n_pos;
	uint32_t n_tokens;
	int H, KV, hd, blk;
	uint8_t* kpool; // this layer's
	uint8_t* vpool;
	const int* table;
	int n_slots, pages_per_seq, n_pages;
	int lanes;      // lanes per head, a power of two >= units / 2 / VP
	int chunk;      // heads per group
	int chunks;     // groups per token
};

// VP: unit pairs per lane (1, or 2 for rows of more than 32 unit pairs)
template <typename T, int VP>
__global__ void __launch_bounds__(kQnThreads) k_qk_norm_rope_rows(const QkNormRopeArgs a)
{
	constexpr int V = Store<T>::kVec; // elements per unit
	pdl_wait();
	pdl_trigger();
	const uint64_t thread = (uint64_t)blockIdx.x * kQnThreads + threadIdx.x;
	const uint64_t group = thread / (uint32_t)a.lanes;
	const int gl = (int)(thread % (uint32_t)a.lanes);
	const uint64_t token = group / (uint32_t)a.chunks;
	// the shuffles below name the whole warp: no thread leaves before the end
	bool on = token < a.n_tokens;
	const int slot = on ? a.tok_slot[token] : -1;
	const int pos = on ? a.tok_pos[token] : 0;
	on = on && slot >= 0; // a negative slot is padding
	const int page_i = on ? pos / a.blk : 0;
	if (on && (slot >= a.n_slots || pos < 0 || pos >= a.n_pos || page_i >= a.pages_per_seq)) {
		if (gl == 0) report_err(a.status, kDevKvRange);
		on = false;
	}
	const int heads = a.H + 2 * a.KV;
	const int h0 = (int)(group % (uint32_t)a.chunks) * a.chunk, h1 = min(heads, h0 + a.chunk);
	const bool writes = on && h1 > a.H;
	const int page = writes ? a.table[(size_t)slot * a.pages_per_seq + page_i] : 0;
	const bool page_ok = page >= 0 && page < a.n_pages;
	if (writes && !page_ok && gl == 0) report_err(a.status, kDevKvRange);
	const int half_units = a.hd / V / 2, half = a.hd / 2;
	float c[VP][V], s[VP][V];
	bool mine[VP];
#pragma unroll
	for (int p = 0; p < VP; ++p) {
		const int u = gl + p * a.lanes;
		mine[p] = on && u < half_units;
#pragma unroll
		for (int i = 0; i < V; i += 4) {
			float4 cc = make_float4(1.f, 1.f, 1.f, 1.f), ss = make_float4(0.f, 0.f, 0.f, 0.f);
			if (mine[p]) {
				cc = *reinterpret_cast<const float4*>(a.rope_cos + (size_t)pos * half + u * V + i);
				ss = *reinterpret_cast<const float4*>(a.rope_sin + (size_t)pos * half + u * V + i);
			}
			c[p][i] = cc.x; c[p][i + 1] = cc.y; c[p][i + 2] = cc.z; c[p][i + 3] = cc.w;
			s[p][i] = ss.x; s[p][i + 1] = ss.y; s[p][i + 2] = ss.z; s[p][i + 3] = ss.w;
		}
	}
	const uint8_t* row = a.qkv + token * a.qkv_stride;
	const uint32_t head_bytes = (uint32_t)a.hd * sizeof(T);
	const uint64_t slab = ((uint64_t)page * a.KV * a.blk + pos % a.blk) * head_bytes; // head 0's row of the page
	for (int hb = h0; hb < h0 + a.chunk; hb += kQnBatch) { // the same trips in every group
		uint4 lo[kQnBatch][VP], hi[kQnBatch][VP];
#pragma unroll
		for (int b = 0; b < kQnBatch; ++b)
#pragma unroll
			for (int p = 0; p < VP; ++p) {
				lo[b][p] = hi[b][p] = make_uint4(0, 0, 0, 0);
				if (mine[p] && hb + b < h1) {
					const uint4* src = reinterpret_cast<const uint4*>(row + (size_t)(hb + b) * head_bytes);
					lo[b][p] = src[gl + p * a.lanes];
					hi[b][p] = src[gl + p * a.lanes + half_units];
				}
			}
#pragma unroll
		for (int b = 0; b < kQnBatch; ++b) {
			const int h = hb + b;
			const bool is_q = h < a.H, is_v = h >= a.H + a.KV;
			float x[VP][V], y[VP][V];
			float ss = 0.0f;
#pragma unroll
			for (int p = 0; p < VP; ++p) {
				unpack_unit(lo[b][p], x[p], (const T*)nullptr);
				unpack_unit(hi[b][p], y[p], (const T*)nullptr);
#pragma unroll
				for (int i = 0; i < V; ++i) ss = fmaf(x[p][i], x[p][i], fmaf(y[p][i], y[p][i], ss));
			}
			for (int o = a.lanes >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
			if (h >= h1) continue;
			if (!is_v) {
				const T* gain = reinterpret_cast<const T*>(is_q ? a.q_gain : a.k_gain);
				const float inv = gain ? 1.0f / sqrtf(ss / (float)a.hd + a.eps) : 1.0f;
#pragma unroll
				for (int p = 0; p < VP; ++p) {
					if (!mine[p]) continue;
					const int u = gl + p * a.lanes;
					if (gain) {
						float g0[V], g1[V];
						unpack_unit(reinterpret_cast<const uint4*>(gain)[u], g0, (const T*)nullptr);
						unpack_unit(reinterpret_cast<const uint4*>(gain)[u + half_units], g1, (const T*)nullptr);
#pragma unroll
						for (int i = 0; i < V; ++i) {
							x[p][i] = x[p][i] * inv * (a.gain_offset + g0[i]);
							y[p][i] = y[p][i] * inv * (a.gain_offset + g1[i]);
						}
					}
					float r0[V], r1[V];
#pragma unroll
					for (int i = 0; i < V; ++i) {
						r0[i] = x[p][i] * c[p][i] - y[p][i] * s[p][i];
						r1[i] = y[p][i] * c[p][i] + x[p][i] * s[p][i];
					}
					lo[b][p] = pack_unit(r0, (T*)nullptr);
					hi[b][p] = pack_unit(r1, (T*)nullptr);
				}
			}
			uint8_t* dst;
			if (is_q) {
				dst = a.q_out + token * a.q_out_stride + (size_t)h * head_bytes;
			} else {
				if (!page_ok) continue;
				const int kvh = h - a.H - (is_v ? a.KV : 0);
				dst = (is_v ? a.vpool : a.kpool) + slab + (uint64_t)kvh * a.blk * head_bytes;
			}
#pragma unroll
			for (int p = 0; p < VP; ++p) {
				if (!mine[p]) continue;
				reinterpret_cast<uint4*>(dst)[gl + p * a.lanes] = lo[b][p];
				reinterpret_cast<uint4*>(dst)[gl + p * a.lanes + half_units] = hi[b][p];
			}
		}
	}
}

} // namespace inf
