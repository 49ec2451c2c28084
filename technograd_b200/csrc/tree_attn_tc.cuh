// tree_attn_tc.cuh -- attention of drafted tokens over a paged cache on tcgen05, for many query rows
// (drafted tokens x heads of a key head's group) and 16-bit caches.
//
// The 128 rows of a unit's tile (k_tree_attn's unit, shares and partial results, tree_attn.cuh) are
// the M of both products, 128 keys a tile: S = Q K^T into one of two TMEM score buffers, P in
// shared memory, O += P V in TMEM. Warps:
//   0-3   softmax, a query row per thread (TMEM lane = row): the running reference mr, p = 2^(z - mr)
//         to P; where a score exceeds mr by more than RAISE, O is rescaled in TMEM, which is rare
//         after the first tiles. At a unit's end the thread holds its row's O, l and mr.
//   4     issue of the MMAs, each as soon as its operands are there: S of the next tile overlaps the
//         softmax of this one.
//   5-12  fetching, two warps each for K and V of even and of odd tiles: rows come by 16-byte
//         cp.async through the page table into the 128-byte-swizzled operand layout (K rows = N,
//         K-major; V rows = the product's k, so V is read MN-major). Pages of any size and stride
//         are thus alike, which TMA boxes of a page would not give. A tile's stage is signalled
//         when it has landed, apart from when the next is asked for.
// What bounds it: with up to 128 rows the cache's bytes (a 64 KB tile pair takes 2850 cycles of the
// measured HBM rate; its MMAs about 2000, its softmax 1300). Every wait is bounded (tc.cuh): a
// timeout sets the status word and all roles leave.
#pragma once

#include <type_traits>

#include "tc.cuh"
#include "tree_attn.cuh"

namespace tgc {

struct TaBars {
	uint64_t kfull[2], kfree[2], vfull[2], vfree[2], s_full[2], s_free[2], p_full, p_empty, done;
	uint32_t tmem;
	int abort;
	int odd[4][2]; // drafted tile: a V row held something not finite (tile & 3; half of its rows)
	long long scan[16];
};

template <int DP> struct TaTile {
	static constexpr int TK = 128, RT = 128, THREADS = 416, NW = 13, CH = DP / 8;
	static constexpr int OP = 128 * DP * 2;                               // bytes of a Q, K or V tile
	static constexpr int Q = 0, K = OP, V = 3 * OP, P = 5 * OP, BARS = P + 128 * 128 * 2;
	static constexpr int SMEM = BARS + (int)sizeof(TaBars);
	static constexpr int SLOT = RT * DP + 2 * RT;
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
__global__ void __launch_bounds__(416, 1) k_tree_attn_tc(const AttnArgs p)
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
			mbar_init(&B->kfree[i], 1), mbar_init(&B->vfree[i], 1);
			mbar_init(&B->s_full[i], 1), mbar_init(&B->s_free[i], 4);
		}
		mbar_init(&B->p_full, 4), mbar_init(&B->p_empty, 1), mbar_init(&B->done, 1);
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
	if (warp == 4) tmem_alloc(&B->tmem, 512); // S buffers at columns 0 and 128, O at 256
	tc_fence_before();
	__syncthreads();
	tc_fence_after();
	const uint32_t tmem = B->tmem;

	if (warp > 4) {
		// ---------------- fetching ----------------
		const int role = warp - 5, isv = role & 1, par = role >> 1 & 1, half = role >> 2;
		uint64_t *full = isv ? &B->vfull[par] : &B->kfull[par], *free_ = isv ? &B->vfree[par] : &B->kfree[par];
		uint8_t *dst = sm + (isv ? A::V : A::K) + par * A::OP;
		const uint32_t sd = smem_u32(dst), sq = smem_u32(sm + A::Q);
		for (int j = 0; j < left; j++, cursor_next<TK>(p, c, 1)) {
			if ((j & 1) != par) continue;
			const bool drafted = c.tile >= c.ctx;
			const char *base = drafted ? (isv ? p.d.v : p.d.k) + (long long)c.b * p.d.kv_seq + c.h * p.d.kv_head : (isv ? p.c.v : p.c.k) + c.h * p.c.head_b;
			// lane's rows half * 64 + lane and + 32 more
			long long at[2];
#pragma unroll
			for (int i = 0; i < 2; i++) {
				const long long x = (long long)(drafted ? 0 : c.tile) * TK + half * 64 + i * 32 + lane;
				if (drafted) at[i] = x < p.d.drafted(c.b) ? x * p.d.kv_tok : -1;
				else at[i] = x < c.n ? p.c.row(p.c.table + (long long)c.b * p.c.cols, (int)x) : -1;
			}
			if (j >= 2 && !ta_wait(B, free_, ((j >> 1) - 1) & 1, p.c)) break;
#pragma unroll
			for (int i = 0; i < 2; i++)
#pragma unroll 8
				for (int y = 0; y < CH; y++) { // 32 / CH rows an instruction
					const int z = y * 32 + lane, r = z / CH, ch = z % CH;
					const long long o = __shfl_sync(~0u, at[i], r);
					const bool have = o >= 0 && ch < chunks;
					cp16(sd + ta_at(half * 64 + i * 32 + r, ch), have ? base + o + ch * 16 : p.d.k, have);
				}
			if (!isv && (j == 0 || c.tile == 0)) { // a unit begins: its Q, once the last S of the unit before is done
				if (j > 0 && !ta_wait(B, &B->kfree[(j - 1) & 1], ((j - 1) >> 1) & 1, p.c)) break;
				for (int z = lane; z < 64 * CH; z += 32) {
					const int row = half * 64 + z / CH, ch = z % CH, r = c.r * RT + row, t = r / p.d.group;
					const bool have = r < rows && ch < chunks;
					cp16(sq + ta_at(row, ch), have ? p.d.q + (long long)c.b * p.d.q_seq + (long long)t * p.d.q_tok + (long long)(c.h * p.d.group + r % p.d.group) * p.d.q_head + ch * 16 : p.d.k, have);
				}
			}
			cp_commit();
			cp_wait<0>();
			if (isv && drafted) {
				// a row that some token does not see may hold anything, and 0 * infinity must not reach O: what is not
				// finite is taken out here and put back for the tokens that see it when O is read
				bool odd = false;
#pragma unroll
				for (int i = 0; i < 2; i++)
#pragma unroll
					for (int y = 0; y < CH; y++) {
						const int z = y * 32 + lane;
						uint32_t *w = (uint32_t *)(dst + ta_at(half * 64 + i * 32 + z / CH, z % CH));
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
	} else if (warp == 4) {
		// ---------------- MMA issue ----------------
		if (lane == 0) {
			const uint32_t id = (1u << 4) | (std::is_same<T, __half>::value ? 0u : (1u << 7) | (1u << 10)) | ((uint32_t)(RT >> 4) << 24); // f32 += f16 or bf16 products
			const uint32_t idS = id | ((uint32_t)(TK >> 3) << 17), idO = id | ((uint32_t)(DP >> 3) << 17) | (1u << 16); // V MN-major
			const uint32_t base = smem_u32(sm);
			int ns = 0, npv = 0;
			bool ok = true;
			long long idle0 = clock64();
			for (uint32_t spins = 0; ok && npv < left;) {
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
				if (npv < ns && ta_test(&B->vfull[npv & 1], (npv >> 1) & 1) && ta_test(&B->p_full, npv & 1)) {
					tc_fence_after();
					const uint32_t pa = base + A::P, v = base + A::V + (npv & 1) * A::OP;
					const bool first = npv == 0 || c.tile == 0;
#pragma unroll
					for (int kk = 0; kk < TK / 16; kk++)
						tc_mma_f16(tmem + 256, sw128_kmajor_desc(pa + (kk >> 2) * 16384 + (kk & 3) * 32), ta_mn_desc(v + kk * 2048, 16384), idO,
							   !first || kk > 0);
					tc_commit(&B->p_empty);
					tc_commit(&B->vfree[npv & 1]);
					npv++;
					cursor_next<TK>(p, c, 1);
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
		const int row = tid;
		const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
		const float zs = p.d.scale * 1.4426950408889634f;
		float mr = -INFINITY, l = 0;
		unsigned long long see = 0;
		int cnt = 0;
		bool from_start = true;
		for (int j = 0; j < left; j++) {
			if (j == 0 || c.tile == 0) { // a unit begins, or goes on from the CTA before
				from_start = c.tile == 0;
				cnt = p.d.drafted(c.b);
				const int t = (c.r * RT + row) / p.d.group;
				see = t < cnt ? p.d.sees(c.b, t, cnt) : 0;
				mr = -INFINITY, l = 0;
			}
			const bool fresh = j == 0 || c.tile == 0, drafted = c.tile >= c.ctx;
			// which of the tile's keys count
			uint32_t ok[4] = {~0u, ~0u, ~0u, ~0u};
			const bool masked = drafted || c.tile == c.ctx - 1;
			if (masked) {
				const int n = drafted ? 0 : (int)(c.n - (long long)c.tile * TK);
#pragma unroll
				for (int w = 0; w < 4; w++)
					ok[w] = drafted ? (w == 0 ? (uint32_t)see : w == 1 ? (uint32_t)(see >> 32) : 0u) : n >= 32 * w + 32 ? ~0u : n <= 32 * w ? 0u : (1u << (n - 32 * w)) - 1;
			}
			if (!ta_wait(B, &B->s_full[j & 1], (j >> 1) & 1, p.c)) break;
			tc_fence_after();
			const uint32_t ts = lanes + (j & 1) * TK;
			float v[32], top = -INFINITY;
#pragma unroll
			for (int w = 0; w < 4; w++) {
				tmem_ld32(ts + w * 32, v);
				float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
				if (masked) {
#pragma unroll
					for (int e = 0; e < 32; e++) x[e & 3] = fmaxf(x[e & 3], ok[w] >> e & 1 ? v[e] * zs : -INFINITY);
				} else {
#pragma unroll
					for (int e = 0; e < 32; e++) x[e & 3] = fmaxf(x[e & 3], v[e] * zs);
				}
				top = fmaxf(top, fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
			}
			if (j > 0 && !ta_wait(B, &B->p_empty, (j - 1) & 1, p.c)) break; // P V of the tile before is done
			const bool raise = top > mr + (SHIFT + RAISE);
			const float ref0 = mr;
			if (raise) mr = top - SHIFT;
			const bool scale = raise && ref0 != -INFINITY;
			if (__any_sync(~0u, scale)) {
				const float f = scale ? ex2(ref0 - mr) : 1;
				l *= f;
				if (!fresh) {
					tc_fence_after();
#pragma unroll 1
					for (int w = 0; w < DP / 32; w++) {
						tmem_ld32(lanes + 256 + w * 32, v);
#pragma unroll
						for (int e = 0; e < 32; e++) v[e] *= f;
						tmem_st32(lanes + 256 + w * 32, v);
					}
				}
			}
			const float ref = mr == -INFINITY ? 0 : mr;
			float sum[4] = {0, 0, 0, 0};
#pragma unroll
			for (int w = 0; w < 4; w++) {
				tmem_ld32(ts + w * 32, v);
				if (masked) {
#pragma unroll
					for (int e = 0; e < 32; e++) v[e] = ok[w] >> e & 1 ? ex2(v[e] * zs - ref) : 0;
				} else {
#pragma unroll
					for (int e = 0; e < 32; e++) v[e] = ex2(v[e] * zs - ref);
				}
#pragma unroll
				for (int e = 0; e < 32; e++) sum[e & 3] += v[e];
#pragma unroll
				for (int i = 0; i < 4; i++)
					*(uint4 *)(sm + A::P + ta_at(row, w * 4 + i)) = make_uint4(pack16(v[8 * i], v[8 * i + 1], T()), pack16(v[8 * i + 2], v[8 * i + 3], T()),
												   pack16(v[8 * i + 4], v[8 * i + 5], T()), pack16(v[8 * i + 6], v[8 * i + 7], T()));
			}
			l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
			tc_fence_before();
			fence_async_smem();
			mbar_arrive_warp(&B->s_free[j & 1]);
			mbar_arrive_warp(&B->p_full);

			const bool end = c.tile == c.all - 1;
			if (end || j == left - 1) {
				if (!ta_wait(B, &B->p_empty, j & 1, p.c)) break;
				tc_fence_after();
				const int r = c.r * RT + row, b = c.b, h = c.h;
				const bool complete = end && from_start, odd = drafted && (*(volatile int *)&B->odd[j & 3][0] | *(volatile int *)&B->odd[j & 3][1]);
				float *slot = complete ? nullptr : p.part + (2ll * blockIdx.x + (from_start ? 1 : 0)) * A::SLOT;
#pragma unroll 1
				for (int w = 0; w < DP / 32; w++) {
					tmem_ld32(lanes + 256 + w * 32, v);
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
						else if (r < rows) store_row4<T>(p, b, h, r, w * 32 + e, cnt, y, mr, l);
					}
				}
				if (!complete) slot[RT * DP + row] = mr, slot[RT * DP + RT + row] = l;
				if (!end && from_start && tid == 0) // the unit goes on in the CTAs after this one
					p.split[blockIdx.x] = make_int4(b, h, c.r, (int)((pos + j + (c.all - 1 - c.tile)) / share));
			}
			cursor_next<TK>(p, c, 1);
		}
	}
	tc_fence_before();
	__syncthreads();
	if (warp == 4) {
		tc_fence_after();
		tmem_dealloc(tmem, 512);
	}
}

} // namespace tgc
