// mma_sync.cuh -- warp-level matrix products for the paged attention's small row tiles: 16 rows
// of a query tile against 8 keys (or 8 dimensions of V) from shared memory, in the element type
// of the cache. Rows of shared memory are `pitch` bytes, their 16-byte chunks XORed with the row
// number modulo 8, so that ldmatrix reads and cp.async writes touch every bank once.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "tc.cuh"

namespace tgc {

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a)
{
	asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t a)
{
	asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}

// d += a b: a 16 x 16 (16 x 8 for tf32) row-major fragments, b 16 x 8 (8 x 8) column-major
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16)
{
	asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
		     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
		     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half)
{
	asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
		     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
		     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma8(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
	asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
		     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
		     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// x = hi + lo in tf32's 11 significant bits each: products of two such pairs without lo lo are
// within 2^-21 of the f32 product
__device__ __forceinline__ void tf32_split(uint32_t x, uint32_t &hi, uint32_t &lo)
{
	asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(__uint_as_float(x)));
	asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(lo) : "f"(__uint_as_float(x) - __uint_as_float(hi)));
}

// A tensor core's accumulation truncates, and thousands of keys add that up to 1e-5 of an f32 output: f32 caches
// leave it only a few products and add those to the sums in f32, rounded to nearest.
__device__ __forceinline__ void add4(float (&d)[4], const float (&t)[4]) { d[0] += t[0], d[1] += t[1], d[2] += t[2], d[3] += t[3]; }

__device__ __forceinline__ uint32_t pack16(float a, float b, __nv_bfloat16)
{
	const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
	return *(const uint32_t *)&v;
}
__device__ __forceinline__ uint32_t pack16(float a, float b, __half)
{
	const __half2 v = __floats2half2_rn(a, b);
	return *(const uint32_t *)&v;
}

// 2^x, relative error 2^-22; 0 for -infinity, NaN for NaN
__device__ __forceinline__ float ex2(float x)
{
	float y;
	asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
	return y;
}

// packed f32 arithmetic, two elements an instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c)
{
	unsigned long long d;
	asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(*(unsigned long long *)&a), "l"(*(unsigned long long *)&b), "l"(*(unsigned long long *)&c));
	return *(float2 *)&d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b)
{
	unsigned long long d;
	asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(*(unsigned long long *)&a), "l"(*(unsigned long long *)&b));
	return *(float2 *)&d;
}

__device__ __forceinline__ float2 mul2(float2 a, float2 b)
{
	unsigned long long d;
	asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(*(unsigned long long *)&a), "l"(*(unsigned long long *)&b));
	return *(float2 *)&d;
}

// Two probabilities as 16-bit high and low parts: within 2^-15 of the number (bf16), 2^-21 (f16), so that P V errs by far less than
// the output's rounding. The high part is cut off a little below the number, so that a positive one has positive parts: an
// infinite V element then stays what it is (but f16 has no low part of numbers below 2^-14).
__device__ __forceinline__ void split16(float2 x, uint32_t &hi, uint32_t &lo, __nv_bfloat16)
{
	const float2 y = mul2(x, make_float2(1 - 0x1p-23f, 1 - 0x1p-23f));
	hi = __byte_perm(__float_as_uint(y.x), __float_as_uint(y.y), 0x7632);
	const float2 z = add2(x, make_float2(-__uint_as_float(__float_as_uint(y.x) & 0xffff0000u), -__uint_as_float(__float_as_uint(y.y) & 0xffff0000u)));
	lo = pack16(z.x, z.y, __nv_bfloat16());
}
__device__ __forceinline__ void split16(float2 x, uint32_t &hi, uint32_t &lo, __half)
{
	const float2 y = mul2(x, make_float2(1 - 0x1p-23f, 1 - 0x1p-23f));
	asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(y.y), "f"(y.x));
	const float2 z = fma2(__half22float2(*(const __half2 *)&hi), make_float2(-1, -1), x);
	lo = pack16(z.x, z.y, __half());
}

// 16 bytes from global to shared memory, or 16 zero bytes
__device__ __forceinline__ void cp16(uint32_t dst, const void *src, bool have)
{
	asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(have ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// The low parts of four f32 elements (tf32_split)
__device__ __forceinline__ uint4 tf32_low(uint4 x)
{
	uint32_t hi;
	uint4 lo;
	tf32_split(x.x, hi, lo.x), tf32_split(x.y, hi, lo.y), tf32_split(x.z, hi, lo.z), tf32_split(x.w, hi, lo.w);
	return lo;
}

// S[16 rows x KW keys] += Q K^T over DP dimensions. KW is 16 for 16-bit elements and 8 for f32, whose Q has its low parts `low` bytes on:
// taken once a unit instead of for every tile of keys, they save a third of the products' instructions (840 rows a key head over 8192 shared
// positions 2293 us, 2802 before).
template <class T, int DP, int MT, int NT>
__device__ __forceinline__ void qk_tile(float (&s)[MT][NT][4], uint32_t sq, uint32_t sk, int lane, int low)
{
	constexpr int P = DP * (int)sizeof(T);
	const int l7 = lane & 7, mi = lane >> 3;
	const uint32_t qrow = sq + ((mi & 1) * 8 + l7) * P;
	if constexpr (sizeof(T) == 2) {
		const uint32_t krow = sk + ((mi >> 1) * 8 + l7) * P;
#pragma unroll
		for (int k = 0; k < DP / 16; k++) {
			uint32_t b[4], a[4];
			ldsm4(b, krow + (((2 * k + (mi & 1)) ^ l7) << 4));
#pragma unroll
			for (int m = 0; m < MT; m++) {
				ldsm4(a, qrow + m * 16 * P + (((2 * k + (mi >> 1)) ^ l7) << 4));
				mma16(s[m][0], a, b[0], b[1], T());
				mma16(s[m][1], a, b[2], b[3], T());
			}
		}
	} else {
		const uint32_t krow = sk + l7 * P;
#pragma unroll 4
		for (int k = 0; k < DP / 16; k++) { // 16 dimensions: two products of 8
			uint32_t b[4], bh[4], bl[4];
			ldsm4(b, krow + (((4 * k + mi) ^ l7) << 4));
#pragma unroll
			for (int i = 0; i < 4; i++) tf32_split(b[i], bh[i], bl[i]);
#pragma unroll
			for (int m = 0; m < MT; m++) {
				float t[4] = {0, 0, 0, 0};
#pragma unroll
				for (int e = 0; e < 2; e++) {
					uint32_t a[4], ah[4], al[4];
					const uint32_t at = qrow + m * 16 * P + (((4 * k + 2 * e + (mi >> 1)) ^ l7) << 4);
					ldsm4(a, at), ldsm4(al, at + low);
#pragma unroll
					for (int i = 0; i < 4; i++) asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(ah[i]) : "f"(__uint_as_float(a[i])));
					mma8(t, al, bh[2 * e], bh[2 * e + 1]);
					mma8(t, ah, bl[2 * e], bl[2 * e + 1]);
					mma8(t, ah, bh[2 * e], bh[2 * e + 1]);
				}
				add4(s[m][0], t);
			}
		}
	}
}

// q . k of two f32 rows as above, in f32
template <int DP> static __device__ __noinline__ float plain_score(uint32_t sq, int row, uint32_t sk, int key)
{
	constexpr int P = DP * 4;
	float s = 0;
#pragma unroll 1
	for (int c = 0; c < P / 16; c++) {
		float q[4], k[4];
		asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(q[0]), "=f"(q[1]), "=f"(q[2]), "=f"(q[3]) : "r"(sq + row * P + ((c ^ (row & 7)) << 4)) : "memory");
		asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(k[0]), "=f"(k[1]), "=f"(k[2]), "=f"(k[3]) : "r"(sk + key * P + ((c ^ (key & 7)) << 4)) : "memory");
#pragma unroll
		for (int i = 0; i < 4; i++) s = fmaf(q[i], k[i], s);
	}
	return s;
}

// An infinite element makes products of split operands NaN where the score may be an infinity (infinity has no low part, and 0 times
// it is not 0): f32 scores that are NaN are taken again without splitting. sq: the first of S's rows.
template <class T, int DP, int MT, int NT>
__device__ __forceinline__ void unsplit_scores(float (&s)[MT][NT][4], uint32_t sq, uint32_t sk, int lane)
{
	if constexpr (sizeof(T) == 4) {
		bool nan = false;
#pragma unroll
		for (int m = 0; m < MT; m++)
#pragma unroll
			for (int x = 0; x < NT; x++)
#pragma unroll
				for (int e = 0; e < 4; e++) nan |= isnan(s[m][x][e]);
		if (!__any_sync(~0u, nan)) return;
#pragma unroll
		for (int m = 0; m < MT; m++)
#pragma unroll
			for (int x = 0; x < NT; x++)
#pragma unroll
				for (int e = 0; e < 4; e++)
					if (isnan(s[m][x][e])) s[m][x][e] = plain_score<DP>(sq, m * 16 + (e >> 1) * 8 + (lane >> 2), sk, x * 8 + 2 * (lane & 3) + (e & 1));
	}
}

// A tile of KW keys as the operand of Q K^T, in registers: for many query rows, which then each
// take their own loads only. f32: hi and lo parts.
template <class T, int DP> struct KeyFrag { uint32_t r[DP / 16][sizeof(T) == 2 ? 4 : 8]; };

template <class T, int DP>
__device__ __forceinline__ void load_keys(KeyFrag<T, DP> &f, uint32_t sk, int lane)
{
	constexpr int P = DP * (int)sizeof(T);
	const int l7 = lane & 7, mi = lane >> 3;
#pragma unroll
	for (int k = 0; k < DP / 16; k++) {
		if constexpr (sizeof(T) == 2) ldsm4(f.r[k], sk + ((mi >> 1) * 8 + l7) * P + (((2 * k + (mi & 1)) ^ l7) << 4));
		else {
			uint32_t b[4];
			ldsm4(b, sk + l7 * P + (((4 * k + mi) ^ l7) << 4));
#pragma unroll
			for (int i = 0; i < 4; i++) tf32_split(b[i], f.r[k][i], f.r[k][4 + i]);
		}
	}
}

// S[MT x 16 rows, KW keys] = Q K^T, Q's rows from sq on; the MT tiles' products are independent
template <class T, int DP, int MT, int NT>
__device__ __forceinline__ void qk_keys(float (&s)[MT][NT][4], const KeyFrag<T, DP> &f, uint32_t sq, int lane)
{
	constexpr int P = DP * (int)sizeof(T);
	const int l7 = lane & 7, mi = lane >> 3;
	const uint32_t qrow = sq + ((mi & 1) * 8 + l7) * P;
#pragma unroll
	for (int m = 0; m < MT; m++)
#pragma unroll
		for (int x = 0; x < NT; x++) s[m][x][0] = s[m][x][1] = s[m][x][2] = s[m][x][3] = 0;
	float whole[MT][NT][4] = {}; // 64 dimensions of 16 bits at a time
#pragma unroll
	for (int k = 0; k < DP / 16; k++) {
		if constexpr (sizeof(T) == 2) {
			uint32_t a[MT][4];
#pragma unroll
			for (int m = 0; m < MT; m++) ldsm4(a[m], qrow + m * 16 * P + (((2 * k + (mi >> 1)) ^ l7) << 4));
			if (DP > 64 && k && k % 4 == 0) { // see add4: a weight is an f32 output
#pragma unroll
				for (int m = 0; m < MT; m++)
#pragma unroll
					for (int x = 0; x < NT; x++)
#pragma unroll
						for (int i = 0; i < 4; i++) whole[m][x][i] += s[m][x][i], s[m][x][i] = 0;
			}
#pragma unroll
			for (int m = 0; m < MT; m++) {
				mma16(s[m][0], a[m], f.r[k][0], f.r[k][1], T());
				mma16(s[m][1], a[m], f.r[k][2], f.r[k][3], T());
			}
		} else {
#pragma unroll
			for (int m = 0; m < MT; m++) {
				float t[4] = {0, 0, 0, 0};
#pragma unroll
				for (int e = 0; e < 2; e++) {
					uint32_t a[4], ah[4], al[4];
					ldsm4(a, qrow + m * 16 * P + (((4 * k + 2 * e + (mi >> 1)) ^ l7) << 4));
#pragma unroll
					for (int i = 0; i < 4; i++) tf32_split(a[i], ah[i], al[i]);
					mma8(t, al, f.r[k][2 * e], f.r[k][2 * e + 1]);
					mma8(t, ah, f.r[k][4 + 2 * e], f.r[k][4 + 2 * e + 1]);
					mma8(t, ah, f.r[k][2 * e], f.r[k][2 * e + 1]);
				}
				add4(s[m][0], t);
			}
		}
	}
	if constexpr (sizeof(T) == 2 && DP > 64) {
#pragma unroll
		for (int m = 0; m < MT; m++)
#pragma unroll
			for (int x = 0; x < NT; x++) add4(s[m][x], whole[m][x]);
	}
}

// O[16 rows x DP] += P V, P in the accumulator layout of qk_tile, 16 bits in two parts (split16). twin: rows 8 to 15 are rows 0 to 7
// again, and take the low parts: the two halves of O add up to theirs.
template <class T, int DP, int MT, int NT>
__device__ __forceinline__ void pv_tile(float (&o)[MT][DP / 8][4], const float (&s)[MT][NT][4], uint32_t sv, int lane, bool twin)
{
	constexpr int P = DP * (int)sizeof(T);
	if constexpr (sizeof(T) == 2) {
		const int l7 = lane & 7, mi = lane >> 3;
		const uint32_t vrow = sv + ((mi & 1) * 8 + l7) * P;
		uint32_t a[MT][4], lo[MT][4];
#pragma unroll
		for (int m = 0; m < MT; m++)
#pragma unroll
			for (int i = 0; i < 4; i++) split16(make_float2(s[m][i >> 1][(i & 1) * 2], s[m][i >> 1][(i & 1) * 2 + 1]), a[m][i], lo[m][i], T());
		if (twin) a[0][1] = lo[0][0], a[0][3] = lo[0][2];
#pragma unroll
		for (int d = 0; d < DP / 16; d++) {
			uint32_t b[4];
			ldsm4t(b, vrow + (((2 * d + (mi >> 1)) ^ l7) << 4));
#pragma unroll
			for (int m = 0; m < MT; m++) {
				mma16(o[m][2 * d], a[m], b[0], b[1], T());
				mma16(o[m][2 * d + 1], a[m], b[2], b[3], T());
			}
			if (!twin) {
#pragma unroll
				for (int m = 0; m < MT; m++) {
					mma16(o[m][2 * d], lo[m], b[0], b[1], T());
					mma16(o[m][2 * d + 1], lo[m], b[2], b[3], T());
				}
			}
		}
	} else {
		// the product's k index runs over keys 0,2,4,6,1,3,5,7: a lane's accumulators are then its operands
		const int g = lane >> 2, t = lane & 3;
		uint32_t ah[MT][4], al[MT][4];
#pragma unroll
		for (int m = 0; m < MT; m++)
#pragma unroll
			for (int i = 0; i < 4; i++) tf32_split(__float_as_uint(s[m][0][(i & 1) * 2 + (i >> 1)]), ah[m][i], al[m][i]);
#pragma unroll
		for (int d = 0; d < DP / 8; d++) {
			const int c = 2 * d + (g >> 2);
			uint32_t b0, b1, h0, l0, h1, l1;
			const uint32_t a0 = sv + 2 * t * P + ((c ^ (2 * t)) << 4) + (g & 3) * 4, a1 = sv + (2 * t + 1) * P + ((c ^ (2 * t + 1)) << 4) + (g & 3) * 4;
			asm volatile("ld.shared.b32 %0, [%1];" : "=r"(b0) : "r"(a0) : "memory");
			asm volatile("ld.shared.b32 %0, [%1];" : "=r"(b1) : "r"(a1) : "memory");
			tf32_split(b0, h0, l0), tf32_split(b1, h1, l1);
#pragma unroll
			for (int m = 0; m < MT; m++) {
				float t[4] = {0, 0, 0, 0};
				mma8(t, al[m], h0, h1);
				mma8(t, ah[m], l0, l1);
				mma8(t, ah[m], h0, h1);
				add4(o[m][d], t);
			}
		}
	}
}

} // namespace tgc
