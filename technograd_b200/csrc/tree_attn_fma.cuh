// tree_attn_fma.cuh -- attention of up to eight query rows over a paged f32 cache on the FMA units.
//
// k_tree_attn's units, shares and rings (tree_attn.cuh), with R rows instead of a tensor core's 16: split products
// would take about 1100 instructions for a warp's 8 keys, most of them for rows that are not there, against 400 here,
// and f32 products need no splitting. A warp's scores: lane (g, t) has a quarter of key g's dimensions, every fourth
// 16-byte piece, in pairs by packed FMAs, and two shuffles add the quarters. Its outputs: a lane has DP / 32 of
// the dimensions for all rows and keys.
// What bounds it: latency where the work is small, else the copies' instructions (160 of the 400) and HBM. Measured:
// 8 sequences of up to 1280 positions, 16 query heads over 8 of 128, 22 us against 29 of the split products.
#pragma once

#include <type_traits>

#include "tree_attn.cuh"

namespace tgc {

template <int DP, int R> struct FmaTile {
	static constexpr int KW = 8, TK = 4 * KW, RT = R, P = DP * 4, CH = P / 16;
	static constexpr int STAGE = 2 * KW * P; // also R x DP floats, what the end of a unit needs
	static constexpr int CTAS = DP == 256 ? 1 : 3, NST = 2;
	static constexpr int Q = 0, RING = RT * P, MASK = RING + 4 * NST * STAGE, ML = MASK + RT * 8, SCAN = ML + 4 * RT * 8;
	static constexpr int SMEM = SCAN + 64;
	static constexpr int SLOT = RT * DP + 2 * RT;
};

template <int DP, int R>
__global__ void __launch_bounds__(128, FmaTile<DP, R>::CTAS) k_tree_attn_fma(const AttnArgs p)
{
	using A = FmaTile<DP, R>;
	constexpr int KW = A::KW, TK = A::TK, P = A::P, CH = A::CH, NST = A::NST, NP = DP / 64; // NP: pairs of a lane's dimensions
	constexpr float RAISE = AttnScale<float>::RAISE;
	extern __shared__ __align__(128) char smem[];
	unsigned long long *s_mask = (unsigned long long *)(smem + A::MASK);
	float2 *s_ml = (float2 *)(smem + A::ML);
	const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
	const uint32_t ring = smem_u32(smem) + A::RING + warp * NST * A::STAGE;
	const int extra = (p.d.tokens + TK - 1) / TK, rows = p.d.tokens * p.d.group, chunks = p.c.dim / 4;
	const float zs = p.d.scale * 1.4426950408889634f;
	pdl_launch();
	pdl_wait();
	AttnCursor c;
	long long left, pos, share;
	if (!attn_share<TK, 4>(p, (long long *)(smem + A::SCAN), extra, c, left, pos, share)) return;
	AttnFetch<float, DP, A> f(p, c, left, ring, extra, chunks);
	float2 o[R][NP];
	float mr[R], l[R];
	int cnt = 0, stage = 0;
	bool first = true, from_start = true;
#pragma unroll
	for (int i = 0; i < NST - 1; i++) f.fetch(i);

	for (long long i = 0; i < left; i++) {
		if (first) { // a unit begins here, or goes on from the CTA before
			first = false;
			from_start = c.tile == 0;
			cnt = p.d.drafted(c.b);
			for (int x = tid; x < R * CH; x += 128) {
				const int row = x / CH, ch = x % CH, r = c.r * R + row, t = r / p.d.group;
				float4 v = make_float4(0, 0, 0, 0);
				if (r < rows && ch < chunks)
					v = *(const float4 *)(p.d.q + (long long)c.b * p.d.q_seq + (long long)t * p.d.q_tok + (long long)(c.h * p.d.group + r - t * p.d.group) * p.d.q_head + ch * 16);
				*(float4 *)(smem + row * P + ch * 16) = v;
			}
			if (tid < R) {
				const int t = (c.r * R + tid) / p.d.group;
				s_mask[tid] = t < cnt ? p.d.sees(c.b, t, cnt) : 0;
			}
#pragma unroll
			for (int r = 0; r < R; r++) {
				mr[r] = -INFINITY, l[r] = 0;
#pragma unroll
				for (int x = 0; x < NP; x++) o[r][x] = make_float2(0, 0);
			}
			__syncthreads();
		}
		f.fetch((stage + NST - 1) % NST); // into the stage of the tile before
		cp_wait<NST - 1>();
		__syncwarp();
		char *sk = smem + A::RING + (warp * NST + stage) * A::STAGE, *sv = sk + KW * P;
		const bool drafted = c.tile >= c.ctx;
		// scores: piece y of lane (g, t4) is 4 (y ^ (g & 1)) + t4, so that two rows' pieces lie in different banks
		float2 d[R];
#pragma unroll
		for (int r = 0; r < R; r++) d[r] = make_float2(0, 0);
#pragma unroll 4
		for (int y = 0; y < CH / 4; y++) {
			const int ch = 4 * (y ^ (g & 1)) + t4;
			const float4 k = *(const float4 *)(sk + g * P + ((ch ^ g) << 4));
#pragma unroll
			for (int r = 0; r < R; r++) {
				const float4 q = *(const float4 *)(smem + r * P + ch * 16);
				d[r] = fma2(make_float2(k.x, k.y), make_float2(q.x, q.y), d[r]);
				d[r] = fma2(make_float2(k.z, k.w), make_float2(q.z, q.w), d[r]);
			}
		}
		const long long key = (long long)(drafted ? c.tile - c.ctx : c.tile) * TK + warp * KW + g;
		float s[R];
		bool up = false;
#pragma unroll
		for (int r = 0; r < R; r++) {
			float x = d[r].x + d[r].y;
			x += __shfl_xor_sync(~0u, x, 1);
			x += __shfl_xor_sync(~0u, x, 2);
			s[r] = (drafted ? s_mask[r] >> key & 1 : key < c.n) ? x * zs : -INFINITY;
			up |= s[r] > mr[r] + RAISE;
		}
		if (__any_sync(~0u, up)) { // raise the references
#pragma unroll
			for (int r = 0; r < R; r++) {
				float top = s[r];
#pragma unroll
				for (int m = 4; m < 32; m <<= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, m));
				if (top > mr[r]) {
					const float a = ex2(mr[r] - top);
					mr[r] = top, l[r] *= a;
#pragma unroll
					for (int x = 0; x < NP; x++) o[r][x] = a == 0 ? make_float2(0, 0) : make_float2(o[r][x].x * a, o[r][x].y * a); // (what has lost its weight may be infinite)
				}
			}
		}
#pragma unroll
		for (int r = 0; r < R; r++) l[r] += s[r] = ex2(s[r] - (mr[r] == -INFINITY ? 0 : mr[r])); // nothing seen yet: 2^-infinity
		auto values = [&](auto guard) { // guard: a row that some token does not see may hold anything, 0 times which is not 0
#pragma unroll
			for (int k = 0; k < KW; k++) {
				float2 v[NP];
				if constexpr (NP == 1) v[0] = *(const float2 *)(sv + k * P + (((lane >> 1) ^ k) << 4) + (lane & 1) * 8);
				else {
#pragma unroll
					for (int x = 0; x < NP; x += 2) {
						const float4 y = *(const float4 *)(sv + k * P + (((x * 16 + lane) ^ k) << 4));
						v[x] = make_float2(y.x, y.y), v[x + 1] = make_float2(y.z, y.w);
					}
				}
#pragma unroll
				for (int r = 0; r < R; r++) {
					const float w = __shfl_sync(~0u, s[r], 4 * k);
					if (decltype(guard)::value && w == 0) continue;
#pragma unroll
					for (int x = 0; x < NP; x++) o[r][x] = fma2(v[x], make_float2(w, w), o[r][x]);
				}
			}
		};
		if (drafted) values(std::true_type());
		else values(std::false_type());
		const bool end = c.tile == c.all - 1, last = i == left - 1;
		if (end || last) {
			// ---- the unit's end, or the share's: join the four warps
#pragma unroll
			for (int r = 0; r < R; r++) {
#pragma unroll
				for (int m = 4; m < 32; m <<= 1) l[r] += __shfl_xor_sync(~0u, l[r], m);
				if (lane == 0) s_ml[warp * R + r] = make_float2(mr[r], l[r]);
			}
			__syncthreads();
#pragma unroll
			for (int r = 0; r < R; r++) {
				float top = -INFINITY;
#pragma unroll
				for (int w = 0; w < 4; w++) top = fmaxf(top, s_ml[w * R + r].x);
				const float a = mr[r] == -INFINITY ? 0 : ex2(mr[r] - top);
#pragma unroll
				for (int x = 0; x < NP; x++) // a pair's column: its lane's place in the V row
					*(float2 *)(sk + (r * DP + (NP == 1 ? lane * 2 : (x / 2 * 32 + lane) * 4 + x % 2 * 2)) * 4) = make_float2(a == 0 ? 0 : o[r][x].x * a, a == 0 ? 0 : o[r][x].y * a);
			}
			__syncthreads();
			const bool complete = end && from_start;
			float *slot = complete ? nullptr : p.part + (2ll * blockIdx.x + (from_start ? 1 : 0)) * A::SLOT;
			for (int x = tid; x < R * DP / 4; x += 128) {
				const int r = x / (DP / 4), col = x % (DP / 4) * 4, row = c.r * R + r;
				float top = -INFINITY, sum = 0;
#pragma unroll
				for (int w = 0; w < 4; w++) top = fmaxf(top, s_ml[w * R + r].x);
				float4 v = make_float4(0, 0, 0, 0);
#pragma unroll
				for (int w = 0; w < 4; w++) {
					const float2 ml = s_ml[w * R + r];
					sum += ml.x == -INFINITY ? ml.y : ml.y * ex2(ml.x - top);
					const float4 y = *(const float4 *)(smem + A::RING + (w * NST + stage) * A::STAGE + (r * DP + col) * 4);
					v.x += y.x, v.y += y.y, v.z += y.z, v.w += y.w;
				}
				if (!complete) {
					*(float4 *)(slot + r * DP + col) = v;
					if (col == 0) slot[R * DP + r] = top, slot[R * DP + R + r] = sum;
				} else if (row < rows) {
					const AttnRow to = attn_row(p, c.b, c.h, row, cnt, sum);
					store_row4<float>(p, to, col, v);
					if (col == 0) store_lse(to, top, sum);
				}
			}
			__syncthreads();
			if (from_start && tid == 0) attn_note(p, c, end, pos, share);
			first = true;
		}
		__syncwarp(); // every lane is done with this stage
		stage = (stage + 1) % NST;
		cursor_next<TK>(p, c, extra);
	}
	cp_wait<0>();
}

} // namespace tgc
