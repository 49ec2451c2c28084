// tree_attn_tc.cuh -- attention of drafted tokens over a paged cache on tcgen05, for many query rows
// (drafted tokens x heads of a key head's group) and 16-bit caches.
//
// The 128 rows of a unit's tile (k_tree_attn's unit, shares and partial results, tree_attn.cuh) are the M of both
// products, 128 keys a tile: S = Q K^T into one of two TMEM score buffers; P over S in V's type, a high and a low part
// (split16), the operand of O += P V that comes from TMEM; O in TMEM. The two halves of a tile's keys have a reference, a sum and an O of
// their own, so their softmax warps need nothing of each other before the unit's end. Warps:
//   0-7   softmax, a query row per thread (TMEM lane = row), warps 4-7 for the tile's second 64 keys: the running
//         reference mr, p = 2^(z - mr) to P; where a score exceeds mr by more than RAISE, O is rescaled in TMEM,
//         which is rare after the first tiles. At a unit's end the two halves exchange mr and l, and each
//         joins and writes half of the row's dimensions.
//   8-15  fetching, two warps each for K and V of even and of odd tiles, through the page table into the
//         128-byte-swizzled operand layout (K rows = N, K-major; V rows = the product's k, so V is read MN-major).
//         Pages of 8, 16, 32 or a multiple of 64 rows come by TMA, a box per page or 64 rows of one (BOX); any other
//         page size or stride, the drafted rows, and V's last tile (what is past its end must be zeros) by
//         16-byte cp.async, about 1000 instructions a tile more: the server case below takes 257 us that way.
//         The copies themselves arrive on the stage's barrier when they have landed, so three stages are on
//         their way at once; the issuing thread's proxy fence orders them before the product's reads. A
//         tile's table entries are read before the tile ahead of it is fetched.
//   16-18 issue of the MMAs, one thread each for S and the halves' P V, as soon as the operands are there: S of the
//         next tiles overlaps the softmax of this one. (One thread for all was busy 3200 cycles a tile with its
//         barriers, commits and issues, more than the tile's bytes take.)
// What bounds it: the chain of a tile and the card's power. (A 64 KB tile pair takes 2850 cycles of the measured HBM rate;
// with P in one part, whose outputs had 1.2 to 1.35 times the error, a tile took 3060 to 3140, and the two cases below 212
// and 69 us: of the difference the second product is about 60%.) Of the 608 x 96 registers of the launch the fetching warps
// give 32 each to the softmax warps, which hold 64 scores. Measured: 48 sequences of up to 6001 positions with 64
// drafted tokens (16 query heads over 8, bf16) 213 us in short runs, 250 us in a long one, which draws 993 W
// and runs at 1545 MHz; 131009 positions with 5 tokens of 8 heads per key head (f16) 84 us, 3.2 TB/s. Every wait
// is bounded (tc.cuh): a timeout sets the status word and all roles leave.
#pragma once

#include <type_traits>

#include "tc.cuh"
#include "tree_attn.cuh"

namespace tgc {

struct TaBars {
	uint64_t kfull[3], kfree[3], vfull[3], vfree[3]; // by stage
	uint64_t s_full[2], p_full[2][2], p_empty[2][2]; // by the tile's parity (P: by half, then parity)
	uint64_t x_full, o_free, done;                   // per unit: mr and l exchanged, O read
	uint32_t tmem;
	int abort;
	int odd[4][2]; // drafted tile: a V row held something not finite (tile & 3; half of its rows)
	long long scan[24];
	float2 ml[2][128];
};

constexpr int TA_REGS = 96; // per thread at launch: 256 x 128 + 256 x 64 + 96 x 96 after the roles' setmaxnreg

template <int DP> struct TaTile {
	static constexpr int TK = 128, RT = 128, NW = 19, THREADS = 32 * NW, CH = DP / 8;
	static constexpr int OP = 128 * DP * 2; // bytes of a Q, K or V tile
	static constexpr int NST = 3, Q = 0, K = OP, V = (1 + NST) * OP, BARS = (1 + 2 * NST) * OP;
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

// Bounded wait; false after the CTA's abort flag or the cycle budget, which sets it.
template <class BARS>
__device__ __forceinline__ bool ta_poll(BARS *B, uint64_t *bar, uint32_t parity, const PgCache &c)
{
	if (ta_test(bar, parity)) return true;
	const long long t0 = clock64();
	for (uint32_t i = 1;; i++) {
		if (ta_test(bar, parity)) return true;
		if ((i & 63) == 0) {
			if (*(volatile int *)&B->abort) return false;
			if (clock64() - t0 > WAIT_CYCLES) {
				c.report(PG_WAIT);
				*(volatile int *)&B->abort = 1;
				return false;
			}
		}
	}
}
// ... of a whole warp, which leaves together
template <class BARS>
__device__ __forceinline__ bool ta_wait(BARS *B, uint64_t *bar, uint32_t parity, const PgCache &c) { return __all_sync(~0u, ta_poll(B, bar, parity, c)); }

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

__device__ __forceinline__ void ta_st32(uint32_t taddr, const uint32_t (&v)[32])
{
#define R(i) "r"(v[i])
	asm volatile(
		"tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,"
		"%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
		R(0), R(1), R(2), R(3), R(4), R(5), R(6), R(7), R(8), R(9), R(10), R(11), R(12), R(13), R(14), R(15), R(16), R(17), R(18), R(19),
		R(20), R(21), R(22), R(23), R(24), R(25), R(26), R(27), R(28), R(29), R(30), R(31)
		: "memory");
#undef R
	asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// D[tmem] (+)= A[tmem] B[smem], A 128 rows (lanes) of 16-bit pairs (columns)
__device__ __forceinline__ void ta_mma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate)
{
	asm volatile(
		"{\n\t.reg .pred p;\n\t"
		"setp.ne.b32 p, %4, 0;\n\t"
		"tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d), "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
		: "memory");
}

// Box of a 4D map into shared memory, its bytes counted on bar; x a multiple of 8, places outside the map are zeros
__device__ __forceinline__ void ta_box(uint32_t dst, const CUtensorMap *map, uint64_t *bar, int x, int c1, int c2, int c3)
{
	asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
		     "l"((uint64_t)map), "r"(smem_u32(bar)), "r"(x), "r"(c1), "r"(c2), "r"(c3)
		     : "memory");
}
__device__ __forceinline__ void ta_expect(uint64_t *bar, uint32_t bytes)
{
	asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}

// An arrival of this thread on bar (counted in its initial count) once all its cp.async copies so far have landed
__device__ __forceinline__ void cp_arrive(uint64_t *bar)
{
	asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// MN-major operand, 128-byte swizzle: rows of 64 elements along MN, 8 rows of k 1024 bytes apart (sbo),
// the next 64 elements of MN lbo bytes on
__device__ __forceinline__ uint64_t ta_mn_desc(uint32_t saddr, uint32_t lbo)
{
	return (uint64_t)((saddr >> 4) & 0x3FFF) | (uint64_t)((lbo >> 4) & 0x3FFF) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

// the largest of three
__device__ __forceinline__ float max3(float a, float b, float c)
{
	float d;
	asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
	return d;
}

// 16-byte chunk c of row r of an operand tile of 128 rows
__device__ __forceinline__ uint32_t ta_at(int r, int c) { return (uint32_t)((c >> 3) * 16384 + r * 128 + (((c & 7) ^ (r & 7)) << 4)); }

// Whether the probability of drafted token u for a query row (token t, head j) is not 0 in f32 against the row's reference
template <class T>
__device__ __forceinline__ bool ta_weighs(const AttnArgs &p, int b, int h, int t, int j, int u, float ref)
{
	const T *q = (const T *)(p.d.q + b * p.d.q_seq + t * p.d.q_tok + j * p.d.q_head);
	const T *k = (const T *)(p.d.k + b * p.d.kv_seq + u * p.d.kv_tok + h * p.d.kv_head);
	float s = 0;
#pragma unroll 1
	for (int i = 0; i < p.c.dim; i++) s = fmaf(PgElem<T>::get(q[i]), PgElem<T>::get(k[i]), s);
	return !(s * p.d.scale * 1.4426950408889634f - ref < -126); // (a score that is NaN counts)
}

template <class T, int DP, bool BOX>
__global__ void __launch_bounds__(608, 1) k_tree_attn_tc(const AttnArgs p, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap)
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
		for (int i = 0; i < A::NST; i++) {
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
		constexpr int RI = 32 / CH;  // rows an instruction copies
		const int ch = lane % CH; // this lane's piece of them
		// its place in a tile: row lane / CH of the warp's half, before the swizzle of the rows after it
		const uint32_t d0 = smem_u32(sm) + (uint32_t)((ch >> 3) * 16384 + (half * 64 + lane / CH) * 128), x0 = (uint32_t)((ch & 7) ^ (lane / CH)) << 4;
		const bool piece = ch < chunks;
		// this lane's rows half * 64 + lane and + 32 more: the table's entries, then the rows' places
		int entry[2], in_page[2];
		uint32_t at[2];
		// by TMA, lane i has box i / (DP / 64) of its half's 64 rows, and 64 of its dimensions
		constexpr int ND = DP / 64;
		const int boxes = BOX ? 64 / p.box.rows : 0;
		auto by_box = [&]() { return BOX && c.tile < c.ctx - isv; };
		auto look = [&]() {
			const bool drafted = c.tile >= c.ctx, box = by_box();
#pragma unroll
			for (int i = 0; i < 2; i++) {
				const int x = (drafted ? 0 : c.tile * TK) + half * 64 + (box ? lane / ND * p.box.rows : i * 32 + lane);
				in_page[i] = -1;
				if (drafted) {
					if (x < p.d.drafted(c.b)) in_page[i] = x;
				} else if (x < c.n && !(box && (i || lane >= boxes * ND))) {
					const int page = x / p.c.page;
					in_page[i] = x - page * p.c.page;
					entry[i] = p.c.table[(long long)c.b * p.c.cols + page];
				}
			}
		};
		if (par < left) {
			if (par) cursor_next<TK>(p, c, 1);
			look();
		}
		int last = -1; // tile asked for
		for (int j = par; j < left; j += 2) {
			const bool drafted = c.tile >= c.ctx, begin = j == 0 || c.tile == 0, box = by_box();
			const int kvh = c.h;
			const int sh = drafted ? 4 : p.c.shift;
			const char *base = (drafted ? (isv ? p.d.v : p.d.k) + (long long)c.b * p.d.kv_seq + c.h * p.d.kv_head : (isv ? p.c.v : p.c.k) + c.h * p.c.head_b) + ch * 16;
			const int st = j % A::NST;
			const char *qb = p.d.q + (long long)c.b * p.d.q_seq + (long long)c.h * p.d.group * p.d.q_head + ch * 16;
			const int r0 = c.r * RT + half * 64 + lane;
#pragma unroll
			for (int i = 0; i < 2; i++)
				at[i] = in_page[i] < 0 ? PG_NONE : box ? (uint32_t)((unsigned)entry[i] < (unsigned)p.c.pages ? in_page[i] : (p.c.report(PG_PAGE), -1)) : drafted ? (uint32_t)(in_page[i] * p.d.kv_tok >> 4) : p.c.at(entry[i], in_page[i]);
			const int page = entry[0];
			if (j + 2 < left) {
				cursor_next<TK>(p, c, 1);
				cursor_next<TK>(p, c, 1);
				look();
			}
			const int tile = (isv ? A::V : A::K) + st * A::OP;
			if (j >= A::NST && !ta_wait(B, isv ? &B->vfree[st] : &B->kfree[st], (j / A::NST - 1) & 1, p.c)) break;
			uint64_t *full = isv ? &B->vfull[st] : &B->kfull[st];
			last = j;
			if (box) {
				if (lane == 0) ta_expect(full, 64 * DP * 2);
				__syncwarp();
				if (lane < boxes * ND) {
					const int r = at[0] == PG_NONE ? 0 : (int)at[0], g = at[0] == PG_NONE ? -1 : page; // -1: zeros
					ta_box(smem_u32(sm) + tile + lane % ND * 16384 + (half * 64 + lane / ND * p.box.rows) * 128, isv ? &vmap : &kmap, full, lane % ND * 64,
					       p.box.swap ? kvh : r, p.box.swap ? r : kvh, g);
				}
			} else
#pragma unroll
			for (int i = 0; i < 2; i++)
#pragma unroll 4
				for (int y = 0; y < CH; y++) {
					const uint32_t o = __shfl_sync(~0u, at[i], y * RI + lane / CH);
					const bool have = o != PG_NONE && piece;
					cp16(d0 + tile + (i * 32 + y * RI) * 128 + (x0 ^ ((y * RI & 7) << 4)), base + ((unsigned long long)(have ? o : 0) << sh), have);
				}
			if (!isv && begin) { // the unit's Q, once the last S of the unit before is done
				if (j > 0 && !ta_wait(B, &B->kfree[(j - 1) % A::NST], (j - 1) / A::NST & 1, p.c)) break;
#pragma unroll 1
				for (int i = 0; i < 2; i++) {
					const int r = r0 + i * 32, t = r / p.d.group;
					const uint32_t mine = r < rows ? (uint32_t)(((long long)t * p.d.q_tok + (long long)(r - t * p.d.group) * p.d.q_head) >> 4) : PG_NONE;
#pragma unroll 4
					for (int y = 0; y < CH; y++) {
						const uint32_t o = __shfl_sync(~0u, mine, y * RI + lane / CH);
						const bool have = o != PG_NONE && piece;
						cp16(d0 + A::Q + (i * 32 + y * RI) * 128 + (x0 ^ ((y * RI & 7) << 4)), qb + ((unsigned long long)(have ? o : 0) << 4), have);
					}
				}
			}
			if (isv && drafted) {
				// a row that some token does not see may hold anything, and 0 * infinity must not reach O: what is not
				// finite is taken out here and put back for the tokens that see it when O is read
				cp_commit();
				cp_wait<0>();
				bool odd = false;
#pragma unroll
				for (int i = 0; i < 2; i++)
#pragma unroll 1
					for (int y = 0; y < CH; y++) {
						uint32_t *w = (uint32_t *)(sm + tile + ta_at(half * 64 + i * 32 + y * RI + lane / CH, ch));
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
				mbar_arrive(full); // of this thread's copies and of what it wrote itself
			} else
				cp_arrive(full);
		}
		cp_commit();
		cp_wait<0>();
		// boxes still on their way land before the CTA's shared memory is released: those of this warp's last
		// tile, and of the one before where no other warp has waited for it
		auto landed = [&](int j) { mbar_wait(isv ? &B->vfull[j % A::NST] : &B->kfull[j % A::NST], j / A::NST & 1, nullptr, 0); };
		if (last >= 0) landed(last);
		if (last >= 2 && last + 1 >= left) landed(last - 2);
	} else if (warp >= 16) {
		// ---------------- MMA issue ----------------
		if (lane == 0) {
			const uint32_t id = (1u << 4) | (std::is_same<T, __half>::value ? 0u : (1u << 7) | (1u << 10)) | ((uint32_t)(RT >> 4) << 24); // f32 += f16 or bf16 products
			const uint32_t base = smem_u32(sm);
			if (warp == 16) {
				const uint32_t idS = id | ((uint32_t)(TK >> 3) << 17), q = base + A::Q;
				for (int j = 0; j < left; j++) {
					// over the P of two tiles before, once that has been used
					if (j >= 2 && (!ta_poll(B, &B->p_empty[0][j & 1], ((j >> 1) - 1) & 1, p.c) || !ta_poll(B, &B->p_empty[1][j & 1], ((j >> 1) - 1) & 1, p.c))) break;
					if (!ta_poll(B, &B->kfull[j % A::NST], j / A::NST & 1, p.c)) break;
					fence_async_smem();
					tc_fence_after();
					const uint32_t k = base + A::K + j % A::NST * A::OP;
#pragma unroll
					for (int kk = 0; kk < DP / 16; kk++)
						tc_mma_f16(tmem + (j & 1) * TK, sw128_kmajor_desc(q + (kk >> 2) * 16384 + (kk & 3) * 32),
							   sw128_kmajor_desc(k + (kk >> 2) * 16384 + (kk & 3) * 32), idS, kk > 0);
					tc_commit(&B->s_full[j & 1]);
					tc_commit(&B->kfree[j % A::NST]);
				}
			} else {
				const int f = warp - 17; // the half of the tile's keys
				const uint32_t idO = id | ((uint32_t)(DP >> 3) << 17) | (1u << 16); // V MN-major
				int unit = 0;
				for (int j = 0; j < left; j++, cursor_next<TK>(p, c, 1)) {
					const bool first = j == 0 || c.tile == 0;
					if (first && unit++ && !ta_poll(B, &B->o_free, unit & 1, p.c)) break; // the unit before has been read
					if (!ta_poll(B, &B->vfull[j % A::NST], j / A::NST & 1, p.c) || !ta_poll(B, &B->p_full[f][j & 1], (j >> 1) & 1, p.c)) break;
					fence_async_smem();
					tc_fence_after();
					const uint32_t pa = tmem + (j & 1) * TK + f * 64, v = base + A::V + j % A::NST * A::OP + f * 8192;
#pragma unroll
					for (int kk = 0; kk < 8; kk++) // P's high parts, then its low ones
						ta_mma_ts(tmem + 256 + f * DP, pa + kk * 8, ta_mn_desc(v + (kk & 3) * 2048, 16384), idO, !first || kk > 0);
					tc_commit(&B->p_empty[f][j & 1]);
					tc_commit(&B->vfree[j % A::NST]);
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
			float mul = zs; // what turns z into the exponent
			if (drafted || c.tile == c.ctx - 1) { // the mask's bits, or the end of the cache
				const int n = drafted ? 0 : (int)(c.n - (long long)c.tile * TK) - hf * 64;
				const unsigned long long ok = drafted ? (hf ? 0ull : see) : n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1;
				const uint32_t lo = (uint32_t)ok, hi = (uint32_t)(ok >> 32);
#pragma unroll
				for (int e = 0; e < 64; e++) z[e] = (e < 32 ? lo : hi) >> (e & 31) & 1 ? z[e] * zs : -INFINITY;
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
				if (!ta_wait(B, &B->p_empty[hf][(j - 1) & 1], ((j - 1) >> 1) & 1, p.c)) break;
				const float f = scale ? ex2(ref0 - mr) : 1;
				l *= f;
				tc_fence_after();
#pragma unroll 1
				for (int w = 0; w < DP / 32; w++) {
					float v[32];
					uint32_t u[32];
					tmem_ld32(mine + w * 32, v);
#pragma unroll
					for (int e = 0; e < 32; e++) u[e] = __float_as_uint(f == 0 ? 0 : v[e] * f);
					ta_st32(mine + w * 32, u);
				}
			}
			const float ref = mr == -INFINITY ? 0 : mr;
			float2 sum[2] = {make_float2(0, 0), make_float2(0, 0)};
			uint32_t pw[32], lo[32];
#pragma unroll
			for (int i = 0; i < 32; i++) {
				const float2 y = fma2(make_float2(z[2 * i], z[2 * i + 1]), make_float2(mul, mul), make_float2(-ref, -ref));
				const float2 q = make_float2(ex2(y.x), ex2(y.y));
				sum[i & 1] = add2(sum[i & 1], q);
				split16(q, pw[i], lo[i], T());
			}
			ta_st32(lanes + (j & 1) * TK + hf * 64, pw); // 64 keys in 32 columns
			ta_st32(lanes + (j & 1) * TK + hf * 64 + 32, lo);
			l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
			tc_fence_before();
			mbar_arrive_warp(&B->p_full[hf][j & 1]);

			const bool end = c.tile == c.all - 1;
			if (end || j == left - 1) {
				// over the unit before's, once the other half has read them too: a unit of one or two tiles needs nothing else of that half
				if (unit && !ta_wait(B, &B->o_free, (unit - 1) & 1, p.c)) break;
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
					if (odd && r < rows && fa != 0) // (the drafted keys are the first half's)
						for (unsigned long long m = see; m; m &= m - 1) {
							const int key = __ffsll((long long)m) - 1, t = r / p.d.group;
							if (!ta_weighs<T>(p, b, h, t, h * p.d.group + (r - t * p.d.group), key, a.x)) continue;
							const T *vr = (const T *)(p.d.v + (long long)b * p.d.kv_seq + (long long)key * p.d.kv_tok + h * p.d.kv_head) + w * 32;
#pragma unroll
							for (int e = 0; e < 32; e++) {
								const float y = w * 32 + e < p.c.dim ? PgElem<T>::get(vr[e]) : 0;
								if (!isfinite(y)) v[e] += y;
							}
						}
					if (!complete) {
#pragma unroll
						for (int e = 0; e < 32; e += 4) *(float4 *)(slot + slot_at<DP, RT>(row, w * 32 + e)) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
					} else if (r < rows) {
#pragma unroll
						for (int e = 0; e < 32; e += 8) store_row8<T>(p, to, w * 32 + e, v + e);
					}
				}
				if (complete && hf == 0 && r < rows) store_lse(to, both, sl);
				if (!complete && hf == 0) slot[RT * DP + row] = both, slot[RT * DP + RT + row] = sl;
				if (from_start && tid == 0) attn_note(p, c, end, pos, share);
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
