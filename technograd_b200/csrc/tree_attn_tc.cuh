// tree_attn_tc.cuh -- attention of drafted tokens over a paged cache on tcgen05, for many query rows
// (drafted tokens x heads of a key head's group) and 16-bit caches.
//
// The 128 rows of a unit's tile (k_tree_attn's unit, shares and partial results, tree_attn.cuh) are
// the M of both products, 128 keys a tile: S = Q K^T into one of two TMEM score buffers, P in
// shared memory, O += P V in TMEM. The two halves of a tile's keys have a reference, a sum and an O
// of their own, so their softmax warps need nothing of each other before the unit's end. Warps:
//   0-7   softmax, a query row per thread (TMEM lane = row), warps 4-7 for the tile's second 64 keys:
//         the running reference mr, p = 2^(z - mr) to P; where a score exceeds mr by more than RAISE,
//         O is rescaled in TMEM, which is rare after the first tiles. At a unit's end the two
//         halves exchange mr and l, and each joins and writes half of the row's dimensions.
//   16    issue of the MMAs, each as soon as its operands are there: S of the next tile overlaps the
//         softmax of this one.
//   8-15  fetching, two warps each for K and V of even and of odd tiles: rows come by 16-byte
//         cp.async through the page table into the 128-byte-swizzled operand layout (K rows = N,
//         K-major; V rows = the product's k, so V is read MN-major). Pages of any size and stride
//         are thus alike, which TMA boxes of a page would not give. A tile's stage is signalled
//         when it has landed, apart from when the next is asked for; the next tile's table entries
//         are looked up while this one's rows are on their way.
// What bounds it: with up to 128 rows the cache's bytes (a 64 KB tile pair takes 2850 cycles of the
// measured HBM rate). Of the 544 x 96 registers of the launch the fetching warps give 32 each to
// the softmax warps, which hold 64 scores. Every wait is bounded (tc.cuh): a timeout sets the status word and all roles
// leave.
#pragma once

#include <type_traits>

#include "tc.cuh"
#include "tree_attn.cuh"

namespace tgc {

struct TaBars {
	uint64_t kfull[2], kfree[2], vfull[2], vfree[2], s_full[2], s_free[2]; // by the tile's parity
	uint64_t p_full[2][2], p_empty[2][2];                                 // by half, then by the tile's parity
	uint64_t x_full, o_free, done;                                        // per unit: mr and l exchanged, O read
	uint32_t tmem;
	int abort;
	int odd[4][2]; // drafted tile: a V row held something not finite (tile & 3; half of its rows)
	long long scan[24];
	float2 ml[2][128];
};

template <int DP> struct TaTile {
	static constexpr int TK = 128, RT = 128, NW = 17, THREADS = 32 * NW, CH = DP / 8;
	static constexpr int OP = 128 * DP * 2;                               // bytes of a Q, K or V tile
	static constexpr int Q = 0, K = OP, V = 3 * OP, P = 5 * OP, PB = 128 * 128 * 2, BARS = P + 2 * PB;
	static constexpr int SMEM = BARS + (int)sizeof(TaBars);
	static constexpr int SLOT = RT * DP + 2 * RT;
	static_assert(SMEM <= 232448, "shared memory of a CTA");
};

__device__ __forceinline__ bool ta_test(uint64_t *bar, uint32_t parity)
{
	uint32_t ok;
	asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
		     : "=r"(ok)
		     : "r"(smem_u32(bar)), "r"(parity)
		     : "memory");
	return ok != 0;
}

// Bounded wait of a whole warp; false after the CTA's abort flag or the cycle budget, which sets it.
__device__ __forceinline__ bool ta_wait(TaBars *B, uint64_t *bar, uint32_t parity, const PgCache &c)
{
	bool ok = true;
	if (!ta_test(bar, parity)) {
		const long long t0 = clock64();
		for (uint32_t i = 1;; i++) {
			if (ta_test(bar, parity)) break;
			if ((i & 63) == 0) {
				if (*(volatile int *)&B->abort) {
					ok = false;
					break;
				}
				if (clock64() - t0 > WAIT_CYCLES) {
					c.report(PG_WAIT);
					*(volatile int *)&B->abort = 1;
					ok = false;
					break;
				}
			}
		}
	}
	return __all_sync(~0u, ok);
}

// 32 lanes x 32 columns of TMEM
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&v)[32])
{
	uint32_t r[32];
	asm volatile(
		"tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
		"%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
		: "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
		  "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
		  "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
		  "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
		: "r"(taddr));
	asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
	for (int i = 0; i < 32; i++) v[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const float (&v)[32])
{
#define R(i) "r"(__float_as_uint(v[i]))
	asm volatile(
		"tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,"
		"%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
		R(0), R(1), R(2), R(3), R(4), R(5), R(6), R(7), R(8), R(9), R(10), R(11), R(12), R(13), R(14), R(15), R(16), R(17), R(18), R(19),
		R(20), R(21), R(22), R(23), R(24), R(25), R(26), R(27), R(28), R(29), R(30), R(31)
		: "memory");
#undef R
	asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// MN-major operand, 128-byte swizzle: rows of 64 elements along MN, 8 rows of k 1024 bytes apart (sbo),
// the next 64 elements of MN lbo bytes on
__device__ __forceinline__ uint64_t ta_mn_desc(uint32_t saddr, uint32_t lbo)
{
	return (uint64_t)((saddr >> 4) & 0x3FFF) | (uint64_t)((lbo >> 4) & 0x3FFF) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

// 16-byte chunk c of row r of an operand tile of 128 rows
__device__ __forceinline__ uint32_t ta_at(int r, int c) { return (uint32_t)((c >> 3) * 16384 + r * 128 + (((c & 7) ^ (r & 7)) << 4)); }

template <class T, int DP>
__global__ void __launch_bounds__(544, 1) k_tree_attn_tc(const AttnArgs p)
{
	using A = TaTile<DP>;
	constexpr int TK = A::TK, RT = A::RT, CH = A::CH;
	constexpr float SHIFT = AttnScale<T>::SHIFT, RAISE = AttnScale<T>::RAISE;
	extern __shared__ __align__(1024) uint8_t ta_raw[];
	uint8_t *sm = ta_raw;
	TaBars *B = (TaBars *)(sm + A::BARS);
	const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
	if (smem_u32(sm) & 1023) { // the operand tiles need 1024-byte alignment
		if (tid == 0) p.c.report(PG_WAIT);
		return;
	}
	if (tid == 0) {
		for (int i = 0; i < 2; i++) {
			mbar_init(&B->kfull[i], 2), mbar_init(&B->vfull[i], 2);
			mbar_init(&B->kfree[i], 1), mbar_init(&B->vfree[i], 2);
			mbar_init(&B->s_full[i], 1), mbar_init(&B->s_free[i], 8);
			for (int k = 0; k < 2; k++) mbar_init(&B->p_full[i][k], 4), mbar_init(&B->p_empty[i][k], 1);
		}
		mbar_init(&B->x_full, 8), mbar_init(&B->o_free, 8), mbar_init(&B->done, 1);
		B->abort = 0;
		fence_barrier_init();
	}
	pdl_launch();
	pdl_wait();
	const int rows = p.d.tokens * p.d.group, chunks = p.c.dim / 8;
	AttnCursor c;
	long long left_, pos, share;
	if (!attn_share<TK, A::NW>(p, B->scan, 1, c, left_, pos, share)) return; // the whole CTA
	const int left = (int)left_;
	if (warp == 16) tmem_alloc(&B->tmem, 512); // S buffers at columns 0 and 128, the halves' O at 256 and 256 + DP
	tc_fence_before();
	__syncthreads();
	tc_fence_after();
	const uint32_t tmem = B->tmem;

	if (warp >= 8 && warp < 16) {
		// ---------------- fetching ----------------
		asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
		const int role = warp - 8, isv = role & 1, par = role >> 1 & 1, half = role >> 2;
		uint64_t *full = isv ? &B->vfull[par] : &B->kfull[par], *free_ = isv ? &B->vfree[par] : &B->kfree[par];
		uint8_t *dst = sm + (isv ? A::V : A::K) + par * A::OP;
		const uint32_t sd = smem_u32(dst), sq = smem_u32(sm + A::Q);
		const int ch = lane % CH; // this lane's piece of the rows it copies
		uint32_t at[2];           // this lane's rows half * 64 + lane and + 32 more: their places, looked up a tile ahead
		auto find = [&]() {
			const bool drafted = c.tile >= c.ctx;
#pragma unroll
			for (int i = 0; i < 2; i++) {
				const int x = (drafted ? 0 : c.tile * TK) + half * 64 + i * 32 + lane;
				at[i] = PG_NONE;
				if (drafted) {
					if (x < p.d.drafted(c.b)) at[i] = (uint32_t)(x * p.d.kv_tok >> 4);
				} else if (x < c.n) {
					const int page = x / p.c.page;
					at[i] = p.c.at(p.c.table[(long long)c.b * p.c.cols + page], x - page * p.c.page);
				}
			}
		};
		if (par < left) {
			if (par) cursor_next<TK>(p, c, 1);
			find();
		}
		for (int j = par; j < left; j += 2) {
			const bool drafted = c.tile >= c.ctx, begin = j == 0 || c.tile == 0;
			const int sh = drafted ? 4 : p.c.shift;
			const char *base = (drafted ? (isv ? p.d.v : p.d.k) + (long long)c.b * p.d.kv_seq + c.h * p.d.kv_head : (isv ? p.c.v : p.c.k) + c.h * p.c.head_b) + ch * 16;
			if (j >= 2 && !ta_wait(B, free_, ((j >> 1) - 1) & 1, p.c)) break;
#pragma unroll
			for (int i = 0; i < 2; i++)
#pragma unroll 8
				for (int y = 0; y < CH; y++) { // 32 / CH rows an instruction
					const int r = y * (32 / CH) + lane / CH;
					const uint32_t o = __shfl_sync(~0u, at[i], r);
					const bool have = o != PG_NONE && ch < chunks;
					cp16(sd + ta_at(half * 64 + i * 32 + r, ch), have ? base + ((unsigned long long)o << sh) : p.d.k, have);
				}
			if (!isv && begin) { // the unit's Q, once the last S of the unit before is done
				if (j > 0 && !ta_wait(B, &B->kfree[(j - 1) & 1], ((j - 1) >> 1) & 1, p.c)) break;
				const char *qb = p.d.q + (long long)c.b * p.d.q_seq + (long long)c.h * p.d.group * p.d.q_head + ch * 16;
#pragma unroll
				for (int i = 0; i < 2; i++) {
					const int r = c.r * RT + half * 64 + i * 32 + lane, t = r / p.d.group;
					const long long mine = r < rows ? (long long)t * p.d.q_tok + (long long)(r - t * p.d.group) * p.d.q_head : -1;
#pragma unroll 4
					for (int y = 0; y < CH; y++) {
						const long long o = __shfl_sync(~0u, mine, y * (32 / CH) + lane / CH);
						const bool have = o >= 0 && ch < chunks;
						cp16(sq + ta_at(half * 64 + i * 32 + y * (32 / CH) + lane / CH, ch), have ? qb + o : p.d.k, have);
					}
				}
			}
			cp_commit();
			if (j + 2 < left) {
				cursor_next<TK>(p, c, 1);
				cursor_next<TK>(p, c, 1);
				find();
			}
			cp_wait<0>();
			if (isv && drafted) {
				// a row that some token does not see may hold anything, and 0 * infinity must not reach O: what is not
				// finite is taken out here and put back for the tokens that see it when O is read
				bool odd = false;
#pragma unroll
				for (int i = 0; i < 2; i++)
#pragma unroll 1
					for (int y = 0; y < CH; y++) {
						uint32_t *w = (uint32_t *)(dst + ta_at(half * 64 + i * 32 + y * (32 / CH) + lane / CH, ch));
#pragma unroll
						for (int x = 0; x < 4; x++)
							if (PgElem<T>::odd(w[x])) {
								odd = true;
								if (PgElem<T>::odd(w[x] & 0xffffu)) w[x] &= 0xffff0000u;
								if (PgElem<T>::odd(w[x] & 0xffff0000u)) w[x] &= 0xffffu;
							}
					}
				odd = __any_sync(~0u, odd);
				if (lane == 0) *(volatile int *)&B->odd[j & 3][half] = odd;
			}
			fence_async_smem();
			mbar_arrive_warp(full);
		}
		cp_wait<0>();
	} else if (warp == 16) {
		// ---------------- MMA issue ----------------
		if (lane == 0) {
			const uint32_t id = (1u << 4) | (std::is_same<T, __half>::value ? 0u : (1u << 7) | (1u << 10)) | ((uint32_t)(RT >> 4) << 24); // f32 += f16 or bf16 products
			const uint32_t idS = id | ((uint32_t)(TK >> 3) << 17), idO = id | ((uint32_t)(DP >> 3) << 17) | (1u << 16); // V MN-major
			const uint32_t base = smem_u32(sm);
			AttnCursor at[2] = {c, c}; // of the halves' next P V
			int ns = 0, npv[2] = {0, 0}, units[2] = {0, 0};
			bool ok = true;
			long long idle0 = clock64();
			for (uint32_t spins = 0; ok && (npv[0] < left || npv[1] < left);) {
				bool did = false;
				if (ns < left && ta_test(&B->kfull[ns & 1], (ns >> 1) & 1) && (ns < 2 || ta_test(&B->s_free[ns & 1], ((ns >> 1) - 1) & 1))) {
					tc_fence_after();
					const uint32_t q = base + A::Q, k = base + A::K + (ns & 1) * A::OP;
#pragma unroll
					for (int kk = 0; kk < DP / 16; kk++)
						tc_mma_f16(tmem + (ns & 1) * TK, sw128_kmajor_desc(q + (kk >> 2) * 16384 + (kk & 3) * 32),
							   sw128_kmajor_desc(k + (kk >> 2) * 16384 + (kk & 3) * 32), idS, kk > 0);
					tc_commit(&B->s_full[ns & 1]);
					tc_commit(&B->kfree[ns & 1]);
					ns++;
					did = true;
				}
#pragma unroll
				for (int f = 0; f < 2; f++) {
					const int j = npv[f];
					if (j >= ns || !ta_test(&B->p_full[f][j & 1], (j >> 1) & 1) || !ta_test(&B->vfull[j & 1], (j >> 1) & 1)) continue;
					const bool first = j == 0 || at[f].tile == 0;
					if (first && j > 0 && !ta_test(&B->o_free, (units[f] - 1) & 1)) continue; // the unit before has been read
					if (first) units[f]++;
					tc_fence_after();
					const uint32_t pa = base + A::P + (j & 1) * A::PB + f * 16384, v = base + A::V + (j & 1) * A::OP + f * 8192;
#pragma unroll
					for (int kk = 0; kk < 4; kk++)
						tc_mma_f16(tmem + 256 + f * DP, sw128_kmajor_desc(pa + kk * 32), ta_mn_desc(v + kk * 2048, 16384), idO, !first || kk > 0);
					tc_commit(&B->p_empty[f][j & 1]);
					tc_commit(&B->vfree[j & 1]);
					npv[f]++;
					cursor_next<TK>(p, at[f], 1);
					did = true;
				}
				if (did) {
					idle0 = clock64(), spins = 0;
				} else if ((++spins & 63) == 0) {
					if (*(volatile int *)&B->abort) ok = false;
					else if (clock64() - idle0 > WAIT_CYCLES) {
						p.c.report(PG_WAIT);
						*(volatile int *)&B->abort = 1;
						ok = false;
					}
				}
			}
			// every MMA issued has completed before TMEM is released (also after an abort)
			tc_commit(&B->done);
			mbar_wait(&B->done, 0, p.c.status + PG_WAIT, 1);
		}
		__syncwarp();
	} else {
		// ---------------- softmax ----------------
		asm volatile("setmaxnreg.inc.sync.aligned.u32 128;");
		const int row = tid & 127, hf = warp >> 2;
		const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16), mine = lanes + 256 + hf * DP;
		const float zs = p.d.scale * 1.4426950408889634f;
		float mr = -INFINITY, l = 0;
		unsigned long long see = 0;
		int cnt = 0, unit = 0;
		bool from_start = true;
		for (int j = 0; j < left; j++) {
			const bool fresh = j == 0 || c.tile == 0, drafted = c.tile >= c.ctx;
			if (fresh) { // a unit begins, or goes on from the CTA before
				from_start = c.tile == 0;
				cnt = p.d.drafted(c.b);
				const int t = (c.r * RT + row) / p.d.group;
				see = t < cnt ? p.d.sees(c.b, t, cnt) : 0;
				mr = -INFINITY, l = 0;
			}
			if (!ta_wait(B, &B->s_full[j & 1], (j >> 1) & 1, p.c)) break;
			tc_fence_after();
			float z[64];
			tmem_ld32(lanes + (j & 1) * TK + hf * 64, *(float (*)[32])z);
			tmem_ld32(lanes + (j & 1) * TK + hf * 64 + 32, *(float (*)[32])(z + 32));
			tc_fence_before();
			mbar_arrive_warp(&B->s_free[j & 1]);
#pragma unroll
			for (int e = 0; e < 64; e++) z[e] *= zs;
			if (drafted || c.tile == c.ctx - 1) { // the mask's bits, or the end of the cache
				const int n = drafted ? 0 : (int)(c.n - (long long)c.tile * TK) - hf * 64;
				const unsigned long long ok = drafted ? (hf ? 0ull : see) : n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1;
				const uint32_t lo = (uint32_t)ok, hi = (uint32_t)(ok >> 32);
#pragma unroll
				for (int e = 0; e < 64; e++)
					if (!((e < 32 ? lo : hi) >> (e & 31) & 1)) z[e] = -INFINITY;
			}
			float x[4] = {z[0], z[1], z[2], z[3]};
#pragma unroll
			for (int e = 4; e < 64; e++) x[e & 3] = fmaxf(x[e & 3], z[e]);
			const float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), ref0 = mr;
			const bool raise = top > mr + (SHIFT + RAISE), scale = raise && ref0 != -INFINITY;
			if (raise) mr = top - SHIFT;
			if (j > 1 && !ta_wait(B, &B->p_empty[hf][j & 1], ((j >> 1) - 1) & 1, p.c)) break; // this P buffer's product is done
			if (__any_sync(~0u, scale)) { // O waits for that of the tile before, too (scale: there is one)
				if (!ta_wait(B, &B->p_empty[hf][(j - 1) & 1], ((j - 1) >> 1) & 1, p.c)) break;
				const float f = scale ? ex2(ref0 - mr) : 1;
				l *= f;
				tc_fence_after();
#pragma unroll 1
				for (int w = 0; w < DP / 32; w++) {
					float v[32];
					tmem_ld32(mine + w * 32, v);
#pragma unroll
					for (int e = 0; e < 32; e++) v[e] *= f;
					tmem_st32(mine + w * 32, v);
				}
			}
			const float ref = mr == -INFINITY ? 0 : mr;
			float sum[4] = {0, 0, 0, 0};
#pragma unroll
			for (int i = 0; i < 8; i++) {
#pragma unroll
				for (int e = 8 * i; e < 8 * i + 8; e++) sum[e & 3] += z[e] = ex2(z[e] - ref);
				*(uint4 *)(sm + A::P + (j & 1) * A::PB + ta_at(row, hf * 8 + i)) = make_uint4(pack16(z[8 * i], z[8 * i + 1], T()), pack16(z[8 * i + 2], z[8 * i + 3], T()),
											pack16(z[8 * i + 4], z[8 * i + 5], T()), pack16(z[8 * i + 6], z[8 * i + 7], T()));
			}
			l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
			tc_fence_before();
			fence_async_smem();
			mbar_arrive_warp(&B->p_full[hf][j & 1]);

			const bool end = c.tile == c.all - 1;
			if (end || j == left - 1) {
				B->ml[hf][row] = make_float2(mr, l);
				mbar_arrive_warp(&B->x_full);
				if (!ta_wait(B, &B->x_full, unit & 1, p.c) || !ta_wait(B, &B->p_empty[0][j & 1], (j >> 1) & 1, p.c) ||
				    !ta_wait(B, &B->p_empty[1][j & 1], (j >> 1) & 1, p.c))
					break;
				tc_fence_after();
				const float2 a = B->ml[0][row], d = B->ml[1][row];
				const float both = fmaxf(a.x, d.x), fa = a.x == -INFINITY ? 0 : ex2(a.x - both), fd = d.x == -INFINITY ? 0 : ex2(d.x - both);
				const float sl = (a.x == -INFINITY ? a.y : a.y * fa) + (d.x == -INFINITY ? d.y : d.y * fd);
				const int r = c.r * RT + row, b = c.b, h = c.h;
				const bool complete = end && from_start, odd = drafted && (*(volatile int *)&B->odd[j & 3][0] | *(volatile int *)&B->odd[j & 3][1]);
				float *slot = complete ? nullptr : p.part + (2ll * blockIdx.x + (from_start ? 1 : 0)) * A::SLOT;
				const AttnRow to = attn_row(p, b, h, r < rows ? r : 0, cnt, sl);
#pragma unroll 1
				for (int w = hf * (DP / 64); w < (hf + 1) * (DP / 64); w++) {
					float v[32], u[32];
					tmem_ld32(lanes + 256 + w * 32, v);
					tmem_ld32(lanes + 256 + DP + w * 32, u);
#pragma unroll
					for (int e = 0; e < 32; e++) v[e] = (fa == 0 ? 0 : v[e] * fa) + (fd == 0 ? 0 : u[e] * fd);
					if (odd && r < rows)
						for (unsigned long long m = see; m; m &= m - 1) {
							const T *vr = (const T *)(p.d.v + (long long)b * p.d.kv_seq + (long long)(__ffsll((long long)m) - 1) * p.d.kv_tok + h * p.d.kv_head) + w * 32;
#pragma unroll
							for (int e = 0; e < 32; e++) {
								const float y = w * 32 + e < p.c.dim ? PgElem<T>::get(vr[e]) : 0;
								if (!isfinite(y)) v[e] += y;
							}
						}
#pragma unroll
					for (int e = 0; e < 32; e += 4) {
						const float4 y = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
						if (!complete) *(float4 *)(slot + row * DP + w * 32 + e) = y;
						else if (r < rows) store_row4<T>(p, to, w * 32 + e, y);
					}
				}
				if (complete && hf == 0 && r < rows) store_lse(to, both, sl);
				if (!complete && hf == 0) slot[RT * DP + row] = both, slot[RT * DP + RT + row] = sl;
				if (!end && from_start && tid == 0) // the unit goes on in the CTAs after this one
					p.split[blockIdx.x] = make_int4(b, h, c.r, (int)((pos + share + (c.all - 2 - c.tile)) / share));
				tc_fence_before();
				mbar_arrive_warp(&B->o_free);
				unit++;
			}
			cursor_next<TK>(p, c, 1);
		}
	}
	tc_fence_before();
	__syncthreads();
	if (warp == 16) {
		tc_fence_after();
		tmem_dealloc(tmem, 512);
	}
}

} // namespace tgc
