// prefix_tc.cuh -- attention over shared prefixes on tcgen05: 16-bit caches of at most 128 dimensions whose pages suit TMA boxes.
//
// tree_attn_tc.cuh's tiles and chain (128 rows by 128 keys, S in two buffers, P in two parts over S, an O for either half of a
// tile's keys) for rows that see every key: no masks, no drafted rows, and a prefix ends where a box does. Fifteen
// warps leave the softmax threads the registers they ask for; within a unit a tile costs no
// look at the list of units. Warps:
//   0-7   softmax, a query row and half of a tile's keys per thread
//   8-11  fetching, two warps each for K (and a unit's Q, by 16-byte cp.async) and V, half a tile's rows each. A box takes the warp
//         that asks for it about 100 cycles: with one warp for all of them pages of 16 rows took 3700 a tile.
//   12-14 issue of the MMAs: S, and the halves' P V. The whole warp waits and counts and one thread issues: eight MMAs take 560
//         cycles so, 1000 where a thread does all by itself.
// What bounds it: with many row tiles the softmax warps' chain, 2560 cycles a tile of which 1024 are exponentials, and the card's power: 1680
// rows a key head over 32768 positions (8 key heads, bf16) 300 us, 590 TFLOP/s. With one, HBM and the asking for boxes: 64 rows over
// 131008 positions (4 key heads, f16, pages of 16) about 60 us, 4.4 TB/s.
#pragma once

#include "tree_attn_tc.cuh"

namespace tgc {

struct PtBars {
	uint64_t kfull[3], kfree[3], vfull[3], vfree[3]; // by stage
	uint64_t s_full[2], p_full[2][2], p_empty[2][2]; // by the tile's parity (P: by half, then parity)
	uint64_t x_full, o_free, done;                   // per unit: mr and l exchanged, O read
	uint32_t tmem;
	int abort;
	long long scan[36];
	AttnCursor begin; // of the CTA's share
	float2 ml[2][128];
};

template <int DP> struct PtTile {
	static constexpr int TK = 128, RT = 128, NW = 15, THREADS = 32 * NW, CH = DP / 8;
	static constexpr int OP = 128 * DP * 2; // bytes of a Q, K or V tile
	static constexpr int NST = 3, Q = 0, K = OP, V = (1 + NST) * OP, BARS = (1 + 2 * NST) * OP;
	static constexpr int SMEM = BARS + (int)sizeof(PtBars);
	static_assert(SMEM <= 232448, "shared memory of a CTA");
};

// ta_wait whose warp sleeps in the barrier between its looks: with fifteen warps looking all the time 40 trees of 21 tokens over 32768
// positions, which run at the card's power limit, took 358 us, so 340.
template <class BARS>
__device__ __forceinline__ bool pt_wait(BARS *B, uint64_t *bar, uint32_t parity, const PgCache &c)
{
	if (__all_sync(~0u, mbar_try(bar, parity))) return true;
	const long long t0 = clock64();
	for (;;) {
		if (__all_sync(~0u, mbar_try(bar, parity))) return true;
		if (__any_sync(~0u, *(volatile int *)&B->abort)) return false;
		if (__any_sync(~0u, clock64() - t0 > WAIT_CYCLES)) {
			c.report(PG_WAIT);
			*(volatile int *)&B->abort = 1;
			return false;
		}
	}
}

// One thread of a warp that is together, always the same
__device__ __forceinline__ bool elect_one()
{
	uint32_t is;
	asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(is));
	return is;
}

// A stage of a ring of three and its parity
struct PtStage {
	int at = 0, parity = 0;
	__device__ __forceinline__ void next()
	{
		if (++at == 3) at = 0, parity ^= 1;
	}
};

template <class T, int DP>
__global__ void __launch_bounds__(480, 1) k_prefix_tc(const SharedArgs p, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap)
{
	using A = PtTile<DP>;
	constexpr int TK = A::TK, RT = A::RT, CH = A::CH, NST = A::NST, MODE = ATTN_PREFIX;
	constexpr float SHIFT = AttnScale<T>::SHIFT, RAISE = AttnScale<T>::RAISE;
	extern __shared__ __align__(1024) uint8_t ta_raw[];
	uint8_t *sm = ta_raw;
	PtBars *B = (PtBars *)(sm + A::BARS);
	static_assert(sizeof(B->scan) / 8 >= 2 * A::NW + 6, "attn_share's words");
	const int tid = threadIdx.x, warp = __shfl_sync(~0u, tid >> 5, 0), lane = tid & 31;
	if (smem_u32(sm) & 1023) { // the operand tiles need 1024-byte alignment
		if (tid == 0) p.c.report(PG_WAIT);
		return;
	}
	if (tid == 0) {
		for (int i = 0; i < NST; i++) {
			mbar_init(&B->kfull[i], 64), mbar_init(&B->vfull[i], 64);
			mbar_init(&B->kfree[i], 1), mbar_init(&B->vfree[i], 2);
		}
		for (int i = 0; i < 2; i++) {
			mbar_init(&B->s_full[i], 1);
			for (int k = 0; k < 2; k++) mbar_init(&B->p_full[i][k], 4), mbar_init(&B->p_empty[i][k], 1);
		}
		mbar_init(&B->x_full, 8), mbar_init(&B->o_free, 8), mbar_init(&B->done, 3);
		B->abort = 0;
		fence_barrier_init();
	}
	shared_begin<MODE>();
	AttnCursor c;
	long long left_, pos, share;
	if (!attn_share<TK, A::NW, MODE, RT>(p, B->scan, 0, c, left_, pos, share)) return; // the whole CTA
	int left = __shfl_sync(~0u, (int)left_, 0);
	// A share that ends one unit and begins another takes the second first: units of one head lie next to each other in the list, so that
	// CTAs at work on them then go through its keys together, from the first on, and most of them find a tile in L2.
	int n1 = 0; // tiles of that second unit
	if (left > c.all - c.tile) {
		AttnCursor next = c;
		next.tile = c.all - 1;
		cursor_next<TK, MODE, RT>(p, next, 0);
		const int rest = left - (c.all - c.tile);
		if (rest <= next.all) {
			if (tid == 0) B->begin = c;
			n1 = rest, c = next;
		}
	}
	if (warp == 12) tmem_alloc(&B->tmem, 512); // S buffers at columns 0 and 128, the halves' O at 256 and 256 + DP
	tc_fence_before();
	__syncthreads();
	tc_fence_after();
	const uint32_t tmem = __shfl_sync(~0u, B->tmem, 0);
	// the tiles of a unit that are this CTA's; then the next unit
	auto here = [&]() { return n1 ? n1 : min(left, c.all - c.tile); };
	auto leave = [&](int n) {
		left -= n;
		if (n1) {
			n1 = 0, c = B->begin;
			return;
		}
		c.tile += n - 1;
		cursor_next<TK, MODE, RT>(p, c, 0);
	};

	if (warp >= 8 && warp < 12) {
		// ---------------- fetching ----------------
		constexpr int RI = 32 / CH, ND = DP / 64; // rows an instruction copies; boxes side by side
		const int isv = warp - 8 >> 1, half = warp & 1, ch = lane % CH, rows_of = p.box.rows, box = half * 64 + lane / ND * rows_of; // this lane's box: its first row
		const bool mine = lane < 64 / rows_of * ND, piece = ch < p.c.dim / 8;
		const uint32_t sm0 = smem_u32(sm), to = sm0 + (isv ? A::V : A::K) + lane % ND * 16384 + box * 128;
		const uint32_t d0 = sm0 + A::Q + (uint32_t)((ch >> 3) * 16384 + (half * 64 + lane / CH) * 128), x0 = (uint32_t)((ch & 7) ^ (lane / CH)) << 4;
		uint64_t *const full = isv ? B->vfull : B->kfull, *const free = isv ? B->vfree : B->kfree;
		PtStage st;
		int j = 0;
		bool ok = true;
		while (left > 0 && ok) {
			const int n = here(), h = c.h;
			const int *table = p.c.table + (long long)c.seq * p.c.cols;
			auto page_of = [&](int tile, int &row) { // of this lane's box of a tile, -1: none
				const int x = tile * TK + box;
				if (!mine || x >= c.n) return -1;
				const int at = x / p.c.page;
				row = x - at * p.c.page;
				return table[at];
			};
			int row = 0, page = page_of(c.tile, row);
			for (int k = 0; k < n; k++, j++) {
				if (page != -1 && (unsigned)page >= (unsigned)p.c.pages) p.c.report(PG_PAGE), page = -1;
				int row1 = 0;
				const int r = page < 0 ? 0 : row, next = k + 1 < n ? page_of(c.tile + k + 1, row1) : -1; // looked up before this tile is waited for
				if (j >= NST && !(ok = pt_wait(B, &free[st.at], st.parity ^ 1, p.c))) break;
				if (lane == 0) ta_expect(&full[st.at], A::OP / 2);
				__syncwarp();
				if (mine) ta_box(to + st.at * A::OP, isv ? &vmap : &kmap, &full[st.at], lane % ND * 64, p.box.swap ? h : r, p.box.swap ? r : h, page < 0 ? -1 : page);
				if (!isv && k == 0) { // the unit's Q, once the last S of the unit before is done
					ok = j == 0 || pt_wait(B, &B->kfree[(j - 1) % NST], (j - 1) / NST & 1, p.c);
					const char *qb = p.d.q + (long long)c.seq * p.d.q_seq + (long long)h * p.d.group * p.d.q_head + ch * 16;
#pragma unroll 1
					for (int i = 0; ok && i < 2; i++) {
						const int x = c.r * RT + half * 64 + i * 32 + lane, t = x / p.d.group, m = t / p.d.tokens;
						const unsigned long long place = x < c.rows ? (unsigned long long)((long long)m * p.d.q_seq + (long long)(t - m * p.d.tokens) * p.d.q_tok + (long long)(x - t * p.d.group) * p.d.q_head) : ~0ull;
#pragma unroll 4
						for (int y = 0; y < CH; y++) {
							const unsigned long long o = __shfl_sync(~0u, place, y * RI + lane / CH);
							const bool have = o != ~0ull && piece;
							cp16(d0 + (i * 32 + y * RI) * 128 + (x0 ^ ((y * RI & 7) << 4)), qb + (have ? o : 0), have);
						}
					}
				}
				cp_arrive(&full[st.at]);
				if (!ok) break;
				st.next();
				page = next, row = row1;
			}
			if (ok) leave(n);
		}
		cp_commit();
		cp_wait<0>();
		// boxes still on their way land before the CTA's shared memory is released (after an abort tile j's may be among them)
		for (int i = max(0, j - NST); i < j + !ok; i++) mbar_wait(&full[i % NST], i / NST & 1, nullptr, 0);
	} else if (warp >= 12) {
		// ---------------- MMA issue ----------------
		const uint32_t id = (1u << 4) | (std::is_same<T, __half>::value ? 0u : (1u << 7) | (1u << 10)) | ((uint32_t)(RT >> 4) << 24); // f32 += f16 or bf16 products
		const uint32_t base = smem_u32(sm);
		PtStage st;
		if (warp == 12) {
			const uint32_t idS = id | ((uint32_t)(TK >> 3) << 17);
			const uint64_t qd = sw128_kmajor_desc(base + A::Q);
			for (int j = 0; j < left; j++, st.next()) {
				// over the P of two tiles before, once that has been used
				if (j >= 2 && (!pt_wait(B, &B->p_empty[0][j & 1], ((j >> 1) - 1) & 1, p.c) || !pt_wait(B, &B->p_empty[1][j & 1], ((j >> 1) - 1) & 1, p.c))) break;
				if (!pt_wait(B, &B->kfull[st.at], st.parity, p.c)) break;
				tc_fence_after();
				if (elect_one()) {
					fence_async_smem();
					const uint64_t kd = sw128_kmajor_desc(base + A::K + st.at * A::OP);
#pragma unroll
					for (int kk = 0; kk < DP / 16; kk++) {
						const uint32_t at = ((kk >> 2) * 16384 + (kk & 3) * 32) >> 4;
						tc_mma_f16(tmem + (j & 1) * TK, qd + at, kd + at, idS, kk > 0);
					}
					tc_commit(&B->s_full[j & 1]);
					tc_commit(&B->kfree[st.at]);
				}
				__syncwarp();
			}
		} else {
			const int f = warp - 13; // the half of the tile's keys
			const uint32_t idO = id | ((uint32_t)(DP >> 3) << 17) | (1u << 16), o = tmem + 256 + f * DP; // V MN-major
			int j = 0, unit = 0;
			bool ok = true;
			while (left > 0 && ok) {
				const int n = here();
				if (unit++ && !pt_wait(B, &B->o_free, unit & 1, p.c)) break; // the unit before has been read
				for (int k = 0; k < n; k++, j++, st.next()) {
					if (!(ok = pt_wait(B, &B->vfull[st.at], st.parity, p.c) && pt_wait(B, &B->p_full[f][j & 1], (j >> 1) & 1, p.c))) break;
					tc_fence_after();
					if (elect_one()) {
						fence_async_smem();
						const uint32_t pa = tmem + (j & 1) * TK + f * 64;
						const uint64_t vd = ta_mn_desc(base + A::V + st.at * A::OP + f * 8192, 16384);
#pragma unroll
						for (int kk = 0; kk < 8; kk++) // 16 keys: P's high parts, then its low ones
							ta_mma_ts(o, pa + (kk >> 1 & 1) * 32 + (kk >> 2) * 16 + (kk & 1) * 8, vd + ((kk & 3) * 2048 >> 4), idO, k > 0 || kk > 0);
						tc_commit(&B->p_empty[f][j & 1]);
						tc_commit(&B->vfree[st.at]);
					}
					__syncwarp();
				}
				if (ok) leave(n);
			}
		}
		// every MMA issued has completed before TMEM is released (also after an abort)
		if (elect_one()) tc_commit(&B->done);
		__syncwarp();
		mbar_wait(&B->done, 0, p.c.status + PG_WAIT, 1);
	} else {
		// ---------------- softmax ----------------
		const int row = tid & 127, hf = warp >> 2;
		const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16), o = lanes + 256 + hf * DP;
		const float zs = p.d.scale * 1.4426950408889634f;
		int j = 0, unit = 0;
		bool ok = true;
		while (left > 0 && ok) {
			const int n = here();
			const bool from_start = c.tile == 0, end = c.tile + n == c.all;
			const int keys = c.n - c.tile * TK - hf * 64; // of this half, from the first tile on
			float mr = -INFINITY, l = 0;
			for (int k = 0; k < n; k++, j++) {
				if (!(ok = pt_wait(B, &B->s_full[j & 1], (j >> 1) & 1, p.c))) break;
				tc_fence_after();
				const uint32_t s = lanes + (j & 1) * TK + hf * 64;
				float z[64];
				tmem_ld32(s, *(float (*)[32])z);
				tmem_ld32(s + 32, *(float (*)[32])(z + 32));
				float mul = zs; // what turns z into the exponent
				const int there = keys - k * TK;
				if (there < 64) { // the prefix ends here
#pragma unroll
					for (int e = 0; e < 64; e++) z[e] = e < there ? z[e] * zs : -INFINITY;
					mul = 1;
				}
				float x[4] = {z[0], z[1], z[2], z[3]}, top;
				if (mul >= 0) {
#pragma unroll
					for (int e = 4; e < 64; e += 2) x[e >> 1 & 3] = max3(x[e >> 1 & 3], z[e], z[e + 1]);
					top = max3(x[0], x[1], fmaxf(x[2], x[3])) * mul;
				} else {
#pragma unroll
					for (int e = 4; e < 64; e++) x[e & 3] = fminf(x[e & 3], z[e]);
					top = fminf(fminf(x[0], x[1]), fminf(x[2], x[3])) * mul;
				}
				const float ref0 = mr;
				const bool raise = top > mr + (SHIFT + RAISE), scale = raise && ref0 != -INFINITY;
				if (raise) mr = top - SHIFT;
				if (__any_sync(~0u, scale)) { // once the product of the tile before is done (scale: there is one)
					if (!(ok = pt_wait(B, &B->p_empty[hf][(j - 1) & 1], ((j - 1) >> 1) & 1, p.c))) break;
					const float by = scale ? ex2(ref0 - mr) : 1;
					l *= by;
					tc_fence_after();
#pragma unroll 1
					for (int w = 0; w < DP / 32; w++) {
						float v[32];
						uint32_t u[32];
						tmem_ld32(o + w * 32, v);
#pragma unroll
						for (int e = 0; e < 32; e++) u[e] = __float_as_uint(by == 0 ? 0 : v[e] * by);
						ta_st32(o + w * 32, u);
					}
				}
				const float ref = mr == -INFINITY ? 0 : mr;
				float2 sum[2] = {make_float2(0, 0), make_float2(0, 0)};
#pragma unroll
				for (int w = 0; w < 2; w++) {
					uint32_t u[32]; // 32 keys: 16 columns of high parts, 16 of low ones
#pragma unroll
					for (int i = 0; i < 16; i++) {
						const float2 y = fma2(make_float2(z[w * 32 + 2 * i], z[w * 32 + 2 * i + 1]), make_float2(mul, mul), make_float2(-ref, -ref));
						const float2 q = make_float2(ex2(y.x), ex2(y.y));
						sum[i & 1] = add2(sum[i & 1], q);
						split16(q, u[i], u[16 + i], T());
					}
					ta_st32(s + w * 32, u);
				}
				l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
				tc_fence_before();
				mbar_arrive_warp(&B->p_full[hf][j & 1]);
			}
			if (!ok) break;
			// the unit's end, or the share's: the two halves join; j is the next tile
			if (unit && !pt_wait(B, &B->o_free, (unit - 1) & 1, p.c)) break; // over the unit before's, once the other half has read them too
			B->ml[hf][row] = make_float2(mr, l);
			mbar_arrive_warp(&B->x_full);
			if (!pt_wait(B, &B->x_full, unit & 1, p.c) || !pt_wait(B, &B->p_empty[0][(j - 1) & 1], ((j - 1) >> 1) & 1, p.c) ||
			    !pt_wait(B, &B->p_empty[1][(j - 1) & 1], ((j - 1) >> 1) & 1, p.c))
				break;
			tc_fence_after();
			const float2 a = B->ml[0][row], d = B->ml[1][row];
			const float both = fmaxf(a.x, d.x), fa = a.x == -INFINITY ? 0 : ex2(a.x - both), fd = d.x == -INFINITY ? 0 : ex2(d.x - both);
			const float sl = (a.x == -INFINITY ? a.y : a.y * fa) + (d.x == -INFINITY ? d.y : d.y * fd);
			const int r = c.r * RT + row;
			const bool complete = end && from_start, there = r < c.rows;
			const long long place = there ? whole_row(p, shared_row<MODE>(p, c, r)) : 0;
			float *slot = p.part + (2ll * blockIdx.x + (from_start ? 1 : 0)) * (RT * (DP + 2));
#pragma unroll 1
			for (int w = hf * (DP / 64); w < (hf + 1) * (DP / 64); w++) {
				float v[32], u[32];
				tmem_ld32(lanes + 256 + w * 32, v);
				tmem_ld32(lanes + 256 + DP + w * 32, u);
#pragma unroll
				for (int e = 0; e < 32; e++) v[e] = (fa == 0 ? 0 : v[e] * fa) + (fd == 0 ? 0 : u[e] * fd);
#pragma unroll
				for (int e = 0; e < 32; e += 4) {
					const float4 y = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
					if (!complete) *(float4 *)(slot + slot_at<DP, RT>(row, w * 32 + e)) = y;
					else if (there) *(float4 *)(p.whole_o + place * DP + w * 32 + e) = y;
				}
			}
			if (hf == 0 && !complete) slot[RT * DP + row] = both, slot[RT * DP + RT + row] = sl;
			else if (hf == 0 && there) p.whole_ml[place] = make_float2(both, sl);
			c.tile += n - 1; // (the part's last tile)
			if (from_start && tid == 0) shared_note<MODE, RT>(p, c, end, pos, share);
			c.tile -= n - 1;
			tc_fence_before();
			mbar_arrive_warp(&B->o_free);
			unit++;
			leave(n);
		}
	}
	tc_fence_before();
	__syncthreads();
	if (warp == 12) {
		tc_fence_after();
		tmem_dealloc(tmem, 512);
	}
}

} // namespace tgc
