/*
 * C ABI of the MI355X (gfx950) data-tiled matmul microkernel library.
 *
 * The first group of entry points keeps the names, argument order, argument
 * meaning, struct layouts and flag values of the reference CPU microkernels in
 * runtime/src/iree/builtins/ukernel so that a caller of those can link against
 * this library unchanged. The second group (prefix iree_uk_mi355x_) has no
 * counterpart in the reference: it exposes what a GPU implementation needs in
 * addition (device selection, stream-ordered launches).
 *
 * Pointer arguments may be host pointers or HIP device pointers. Classification
 * looks only at `buffer + offset` (never at `buffer` itself, which the
 * reference's own tests set to an address before the allocation), see
 * iree_uk_mi355x_set_stream() for the rules.
 *
 * Everything here is plain C: no HIP or torch types appear in a signature.
 */
#ifndef IREE_UK_MI355X_H_
#define IREE_UK_MI355X_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Signed 64-bit index type on 64-bit targets (reference: common.h:269-275). */
typedef long long iree_uk_index_t;

/*===--------------------------------------------------------------------===*/
/* Flag values. Fixed by the reference compiler and runtime sharing them      */
/* (reference: exported_bits.h:29-49, 56-66, 73-83).                          */
/*===--------------------------------------------------------------------===*/

#define IREE_UK_FLAG_MMT4D_TYPE_MASK 0xFF
#define IREE_UK_FLAG_MMT4D_TYPE_NONE 0x00
#define IREE_UK_FLAG_MMT4D_TYPE_F32F32F32 0x01
#define IREE_UK_FLAG_MMT4D_TYPE_S8S8S32 0x02
#define IREE_UK_FLAG_MMT4D_TYPE_F16F16F32 0x03
#define IREE_UK_FLAG_MMT4D_TYPE_F16F16F16 0x04
#define IREE_UK_FLAG_MMT4D_TYPE_BF16BF16F32 0x05
#define IREE_UK_FLAG_MMT4D_TYPE_BF16BF16BF16 0x06
#define IREE_UK_FLAG_MMT4D_TYPE_S16S16S32 0x07
#define IREE_UK_FLAG_MMT4D_TYPE_S16U4S32 0x08
#define IREE_UK_FLAG_MMT4D_TYPE_S16S8S32 0x09
#define IREE_UK_FLAG_MMT4D_TYPE_S8S4S32 0x0A
#define IREE_UK_FLAG_MMT4D_TYPE_END 0x0B
#define IREE_UK_FLAG_MMT4D_ACCUMULATE 0x100
#define IREE_UK_FLAG_MMT4D_ALLOW_GENERIC_FALLBACK_TILE_FUNCTION 0x200
#define IREE_UK_FLAG_MMT4D_SKIP_INTERMEDIATE_ROUNDINGS 0x400
#define IREE_UK_FLAG_MMT4D_INFO_HAVE_ARCHITECTURE_SPECIFIC_TILE_FUNCTION 0x1

#define IREE_UK_FLAG_PACK_TYPE_MASK 0xFF
#define IREE_UK_FLAG_PACK_TYPE_NONE 0x00
#define IREE_UK_FLAG_PACK_TYPE_F32F32 0x01
#define IREE_UK_FLAG_PACK_TYPE_I8I8 0x02
#define IREE_UK_FLAG_PACK_TYPE_I32I32 0x03
#define IREE_UK_FLAG_PACK_TYPE_F16F16 0x04
#define IREE_UK_FLAG_PACK_TYPE_BF16BF16 0x05
#define IREE_UK_FLAG_PACK_TRANSPOSE_INNER 0x100
#define IREE_UK_FLAG_PACK_TRANSPOSE_OUTER 0x200

#define IREE_UK_FLAG_UNPACK_TYPE_MASK 0xFF
#define IREE_UK_FLAG_UNPACK_TYPE_NONE 0x00
#define IREE_UK_FLAG_UNPACK_TYPE_F32F32 0x01
#define IREE_UK_FLAG_UNPACK_TYPE_I32I32 0x03
#define IREE_UK_FLAG_UNPACK_TYPE_F16F16 0x04
#define IREE_UK_FLAG_UNPACK_TYPE_BF16BF16 0x05
#define IREE_UK_FLAG_UNPACK_TRANSPOSE_INNER 0x100
#define IREE_UK_FLAG_UNPACK_TRANSPOSE_OUTER 0x200

#define IREE_UK_FLAG_QUERY_TILE_SIZES_OPERAND_ROLE_MASK 0xFF
#define IREE_UK_FLAG_QUERY_TILE_SIZES_OPERAND_ROLE_NONE 0x00
#define IREE_UK_FLAG_QUERY_TILE_SIZES_OPERAND_ROLE_LHS 0x01
#define IREE_UK_FLAG_QUERY_TILE_SIZES_OPERAND_ROLE_RHS 0x02
#define IREE_UK_FLAG_QUERY_TILE_SIZES_OPERAND_ROLE_RESULT 0x03
#define IREE_UK_FLAG_QUERY_TILE_SIZES_OPERATION_MASK 0xFF00
#define IREE_UK_FLAG_QUERY_TILE_SIZES_OPERATION_NONE 0x0000
#define IREE_UK_FLAG_QUERY_TILE_SIZES_OPERATION_MATMUL_F32F32F32 0x0100
#define IREE_UK_FLAG_QUERY_TILE_SIZES_OPERATION_MATMUL_I8I8I32 0x0200
#define IREE_UK_FLAG_QUERY_TILE_SIZES_OPERATION_MATMUL_F16F16F32 0x0300
#define IREE_UK_FLAG_QUERY_TILE_SIZES_OPERATION_MATMUL_F16F16F16 0x0400
#define IREE_UK_FLAG_QUERY_TILE_SIZES_OPERATION_MATMUL_BF16BF16F32 0x0500
#define IREE_UK_FLAG_QUERY_TILE_SIZES_OPERATION_MATMUL_BF16BF16BF16 0x0600

/* Flag values of the microscaled operators and of the norm (no counterpart in
 * the reference). Type flags name the input's type, then the output's; of
 * products the lhs, the rhs and the result. E2M1 and E4M3 are the 4-bit and
 * 8-bit floats of the OCP microscaling formats, always with E8M0 scales. */
#define IREE_UK_MI355X_FLAG_MX_PACK_TYPE_MASK 0xFF
#define IREE_UK_MI355X_FLAG_MX_PACK_TYPE_F32E2M1 0x01
#define IREE_UK_MI355X_FLAG_MX_PACK_TYPE_F16E2M1 0x02
#define IREE_UK_MI355X_FLAG_MX_PACK_TYPE_BF16E2M1 0x03
#define IREE_UK_MI355X_FLAG_MX_PACK_TYPE_F32E4M3 0x04
#define IREE_UK_MI355X_FLAG_MX_PACK_TYPE_F16E4M3 0x05
#define IREE_UK_MI355X_FLAG_MX_PACK_TYPE_BF16E4M3 0x06

#define IREE_UK_MI355X_FLAG_MX_UNPACK_TYPE_MASK 0xFF
#define IREE_UK_MI355X_FLAG_MX_UNPACK_TYPE_E2M1F32 0x01
#define IREE_UK_MI355X_FLAG_MX_UNPACK_TYPE_E2M1F16 0x02
#define IREE_UK_MI355X_FLAG_MX_UNPACK_TYPE_E2M1BF16 0x03
#define IREE_UK_MI355X_FLAG_MX_UNPACK_TYPE_E4M3F32 0x04
#define IREE_UK_MI355X_FLAG_MX_UNPACK_TYPE_E4M3F16 0x05
#define IREE_UK_MI355X_FLAG_MX_UNPACK_TYPE_E4M3BF16 0x06

#define IREE_UK_MI355X_FLAG_MX_MMT4D_TYPE_MASK 0xFF
#define IREE_UK_MI355X_FLAG_MX_MMT4D_TYPE_E2M1E2M1F32 0x01
#define IREE_UK_MI355X_FLAG_MX_MMT4D_TYPE_E2M1E2M1F16 0x02
#define IREE_UK_MI355X_FLAG_MX_MMT4D_TYPE_E2M1E2M1BF16 0x03
#define IREE_UK_MI355X_FLAG_MX_MMT4D_TYPE_E4M3E2M1F32 0x04
#define IREE_UK_MI355X_FLAG_MX_MMT4D_TYPE_E4M3E2M1F16 0x05
#define IREE_UK_MI355X_FLAG_MX_MMT4D_TYPE_E4M3E2M1BF16 0x06
#define IREE_UK_MI355X_FLAG_MX_MMT4D_ACCUMULATE 0x100

#define IREE_UK_MI355X_FLAG_RMS_NORM_TYPE_MASK 0xFF
#define IREE_UK_MI355X_FLAG_RMS_NORM_TYPE_F32S8 0x01
#define IREE_UK_MI355X_FLAG_RMS_NORM_TYPE_F16S8 0x02
#define IREE_UK_MI355X_FLAG_RMS_NORM_TYPE_BF16S8 0x03
#define IREE_UK_MI355X_FLAG_RMS_NORM_TYPE_F32E4M3 0x04
#define IREE_UK_MI355X_FLAG_RMS_NORM_TYPE_F16E4M3 0x05
#define IREE_UK_MI355X_FLAG_RMS_NORM_TYPE_BF16E4M3 0x06
#define IREE_UK_MI355X_FLAG_RMS_NORM_TYPE_F32E2M1 0x07
#define IREE_UK_MI355X_FLAG_RMS_NORM_TYPE_F16E2M1 0x08
#define IREE_UK_MI355X_FLAG_RMS_NORM_TYPE_BF16E2M1 0x09
#define IREE_UK_MI355X_FLAG_RMS_NORM_WEIGHT_F32 0x100

/* Flag values of the feed-forward operators (no counterpart in the reference).
 * Type flags name the operands' type twice, then the result's. */
#define IREE_UK_MI355X_FLAG_GATED_MMT4D_TYPE_MASK 0xFF
#define IREE_UK_MI355X_FLAG_GATED_MMT4D_TYPE_F16F16F32 0x01
#define IREE_UK_MI355X_FLAG_GATED_MMT4D_TYPE_F16F16F16 0x02
#define IREE_UK_MI355X_FLAG_GATED_MMT4D_TYPE_BF16BF16F32 0x03
#define IREE_UK_MI355X_FLAG_GATED_MMT4D_TYPE_BF16BF16BF16 0x04
#define IREE_UK_MI355X_FLAG_GATED_MMT4D_ACTIVATION_MASK 0xF00
#define IREE_UK_MI355X_FLAG_GATED_MMT4D_SILU 0x100
#define IREE_UK_MI355X_FLAG_GATED_MMT4D_GELU 0x200
#define IREE_UK_MI355X_FLAG_GATED_MMT4D_SIGMOID 0x300
#define IREE_UK_MI355X_FLAG_GATED_MMT4D_PRE_LOAD 0x1000
#define IREE_UK_MI355X_FLAG_GATED_MMT4D_PRE_STORE 0x2000
#define IREE_UK_MI355X_FLAG_GATED_MMT4D_PRE_F32 0x4000
#define IREE_UK_MI355X_FLAG_GATED_MMT4D_ACCUMULATE 0x8000

#define IREE_UK_MI355X_FLAG_ADAPTER_MMT4D_TYPE_MASK 0xFF
#define IREE_UK_MI355X_FLAG_ADAPTER_MMT4D_TYPE_F16F16F32 0x01
#define IREE_UK_MI355X_FLAG_ADAPTER_MMT4D_TYPE_F16F16F16 0x02
#define IREE_UK_MI355X_FLAG_ADAPTER_MMT4D_TYPE_BF16BF16F32 0x03
#define IREE_UK_MI355X_FLAG_ADAPTER_MMT4D_TYPE_BF16BF16BF16 0x04
#define IREE_UK_MI355X_FLAG_ADAPTER_MMT4D_ACCUMULATE 0x100

/*===--------------------------------------------------------------------===*/
/* Parameter structs (field order and types are ABI).                         */
/*===--------------------------------------------------------------------===*/

/* reference: mmt4d_internal.h:14-32. Offsets and strides count ELEMENTS of the
 * operand's type (4-bit elements included); M, N, K count tiles. Only the
 * outermost dimension of each operand is strided. */
typedef struct iree_uk_mmt4d_params_t {
  const void* lhs_buffer;
  iree_uk_index_t lhs_offset;
  iree_uk_index_t lhs_stride0;
  const void* rhs_buffer;
  iree_uk_index_t rhs_offset;
  iree_uk_index_t rhs_stride0;
  void* out_buffer;
  iree_uk_index_t out_offset;
  iree_uk_index_t out_stride0;
  iree_uk_index_t M;
  iree_uk_index_t N;
  iree_uk_index_t K;
  int32_t M0;
  int32_t N0;
  int32_t K0;
  uint32_t flags;
  const uint64_t* cpu_data;
} iree_uk_mmt4d_params_t;

/* reference: pack_internal.h:12-30. */
typedef struct iree_uk_pack_params_t {
  const void* in_buffer;
  iree_uk_index_t in_offset;
  iree_uk_index_t in_stride0;
  iree_uk_index_t in_stride1;
  void* out_buffer;
  iree_uk_index_t out_offset;
  iree_uk_index_t out_stride0;
  iree_uk_index_t out_stride1;
  iree_uk_index_t in_size0;
  iree_uk_index_t in_size1;
  iree_uk_index_t out_size0;
  iree_uk_index_t out_size1;
  iree_uk_index_t out_size2;
  iree_uk_index_t out_size3;
  uint64_t padding_value;
  uint32_t flags;
  const uint64_t* cpu_data;
} iree_uk_pack_params_t;

/* reference: unpack_internal.h:12-29. */
typedef struct iree_uk_unpack_params_t {
  const void* in_buffer;
  iree_uk_index_t in_offset;
  iree_uk_index_t in_stride0;
  iree_uk_index_t in_stride1;
  void* out_buffer;
  iree_uk_index_t out_offset;
  iree_uk_index_t out_stride0;
  iree_uk_index_t out_stride1;
  iree_uk_index_t in_size0;
  iree_uk_index_t in_size1;
  iree_uk_index_t in_size2;
  iree_uk_index_t in_size3;
  iree_uk_index_t out_size0;
  iree_uk_index_t out_size1;
  uint32_t flags;
  const uint64_t* cpu_data;
} iree_uk_unpack_params_t;

/* reference: query_tile_sizes.h:17-27. */
typedef struct iree_uk_query_tile_sizes_2d_params_t {
  uint32_t flags;
  iree_uk_index_t size0;
  iree_uk_index_t size1;
  const uint64_t* cpu_data;
} iree_uk_query_tile_sizes_2d_params_t;

typedef struct iree_uk_query_tile_sizes_2d_out_params_t {
  iree_uk_index_t tile_size0;
  iree_uk_index_t tile_size1;
} iree_uk_query_tile_sizes_2d_out_params_t;

/* Parameters of the operators without a counterpart in the reference, in the
 * same manner: offsets and strides count ELEMENTS of the buffer's type (4-bit
 * elements included; a scale is an element of one byte), only the outermost
 * dimension of tiled operands is strided. */
typedef struct iree_uk_mi355x_mx_pack_params_t {
  const void* in_buffer;
  iree_uk_index_t in_offset;
  iree_uk_index_t in_stride0;
  iree_uk_index_t in_stride1;
  void* out_buffer;
  iree_uk_index_t out_offset;
  iree_uk_index_t out_stride0;
  void* scales_buffer;
  iree_uk_index_t scales_offset;
  iree_uk_index_t scales_stride0;
  iree_uk_index_t in_size0;
  iree_uk_index_t in_size1;
  iree_uk_index_t out_size0;
  iree_uk_index_t out_size1;
  iree_uk_index_t out_size2;
  iree_uk_index_t out_size3;
  uint32_t flags;
} iree_uk_mi355x_mx_pack_params_t;

typedef struct iree_uk_mi355x_mx_unpack_params_t {
  const void* in_buffer;
  iree_uk_index_t in_offset;
  iree_uk_index_t in_stride0;
  const void* scales_buffer;
  iree_uk_index_t scales_offset;
  iree_uk_index_t scales_stride0;
  void* out_buffer;
  iree_uk_index_t out_offset;
  iree_uk_index_t out_stride0;
  iree_uk_index_t out_stride1;
  iree_uk_index_t in_size0;
  iree_uk_index_t in_size1;
  iree_uk_index_t in_size2;
  iree_uk_index_t in_size3;
  iree_uk_index_t out_size0;
  iree_uk_index_t out_size1;
  uint32_t flags;
} iree_uk_mi355x_mx_unpack_params_t;

typedef struct iree_uk_mi355x_mx_mmt4d_params_t {
  const void* lhs_buffer;
  iree_uk_index_t lhs_offset;
  iree_uk_index_t lhs_stride0;
  const void* lhs_scales_buffer;
  iree_uk_index_t lhs_scales_offset;
  iree_uk_index_t lhs_scales_stride0;
  const void* rhs_buffer;
  iree_uk_index_t rhs_offset;
  iree_uk_index_t rhs_stride0;
  const void* rhs_scales_buffer;
  iree_uk_index_t rhs_scales_offset;
  iree_uk_index_t rhs_scales_stride0;
  void* out_buffer;
  iree_uk_index_t out_offset;
  iree_uk_index_t out_stride0;
  iree_uk_index_t M;
  iree_uk_index_t N;
  iree_uk_index_t K;
  int32_t M0;
  int32_t N0;
  int32_t K0;
  uint32_t flags;
} iree_uk_mi355x_mx_mmt4d_params_t;

typedef struct iree_uk_mi355x_rms_norm_params_t {
  const void* in_buffer;
  iree_uk_index_t in_offset;
  iree_uk_index_t in_stride0;
  const void* residual_buffer; /* NULL: nothing is added */
  iree_uk_index_t residual_offset;
  iree_uk_index_t residual_stride0;
  void* sum_buffer; /* NULL: the sum is not stored */
  iree_uk_index_t sum_offset;
  iree_uk_index_t sum_stride0;
  const void* weight_buffer; /* NULL: ones */
  iree_uk_index_t weight_offset;
  void* out_buffer;
  iree_uk_index_t out_offset;
  iree_uk_index_t out_stride0;
  void* scales_buffer;
  iree_uk_index_t scales_offset;
  iree_uk_index_t scales_stride0;
  iree_uk_index_t size0;
  iree_uk_index_t size1;
  iree_uk_index_t out_size1;
  float epsilon;
  uint32_t flags;
} iree_uk_mi355x_rms_norm_params_t;

typedef struct iree_uk_mi355x_gated_mmt4d_params_t {
  const void* lhs_buffer;
  iree_uk_index_t lhs_offset;
  iree_uk_index_t lhs_stride0;
  const void* gate_buffer;
  iree_uk_index_t gate_offset;
  iree_uk_index_t gate_stride0;
  const void* up_buffer;
  iree_uk_index_t up_offset;
  iree_uk_index_t up_stride0;
  void* gate_pre_buffer; /* with PRE_LOAD or PRE_STORE */
  iree_uk_index_t gate_pre_offset;
  iree_uk_index_t gate_pre_stride0;
  void* up_pre_buffer;
  iree_uk_index_t up_pre_offset;
  iree_uk_index_t up_pre_stride0;
  void* out_buffer;
  iree_uk_index_t out_offset;
  iree_uk_index_t out_stride0;
  iree_uk_index_t M;
  iree_uk_index_t N;
  iree_uk_index_t K;
  int32_t M0;
  int32_t N0;
  int32_t K0;
  uint32_t flags;
} iree_uk_mi355x_gated_mmt4d_params_t;

typedef struct iree_uk_mi355x_gated_mmt4d_backward_params_t {
  const void* lhs_buffer;
  iree_uk_index_t lhs_offset;
  iree_uk_index_t lhs_stride0;
  const void* gate_buffer;
  iree_uk_index_t gate_offset;
  iree_uk_index_t gate_stride0;
  const void* up_buffer;
  iree_uk_index_t up_offset;
  iree_uk_index_t up_stride0;
  const void* gate_pre_buffer;
  iree_uk_index_t gate_pre_offset;
  iree_uk_index_t gate_pre_stride0;
  const void* up_pre_buffer;
  iree_uk_index_t up_pre_offset;
  iree_uk_index_t up_pre_stride0;
  const void* out_grad_buffer;
  iree_uk_index_t out_grad_offset;
  iree_uk_index_t out_grad_stride0;
  void* lhs_grad_buffer; /* NULL: not computed */
  iree_uk_index_t lhs_grad_offset;
  iree_uk_index_t lhs_grad_stride0;
  void* gate_grad_buffer; /* NULL: not computed */
  iree_uk_index_t gate_grad_offset;
  iree_uk_index_t gate_grad_stride0;
  void* up_grad_buffer; /* NULL: not computed */
  iree_uk_index_t up_grad_offset;
  iree_uk_index_t up_grad_stride0;
  void* workspace_buffer;
  iree_uk_index_t workspace_size; /* bytes */
  iree_uk_index_t M;
  iree_uk_index_t N;
  iree_uk_index_t K;
  int32_t M0;
  int32_t N0;
  int32_t K0;
  uint32_t flags;
} iree_uk_mi355x_gated_mmt4d_backward_params_t;

typedef struct iree_uk_mi355x_adapter_mmt4d_params_t {
  const void* lhs_buffer;
  iree_uk_index_t lhs_offset;
  iree_uk_index_t lhs_stride0;
  const void* down_buffer;
  iree_uk_index_t down_offset;
  iree_uk_index_t down_stride0;
  iree_uk_index_t down_stride1;
  const void* up_buffer;
  iree_uk_index_t up_offset;
  iree_uk_index_t up_stride0;
  iree_uk_index_t up_stride1;
  const int32_t* index_buffer;
  iree_uk_index_t index_offset;
  const float* scales_buffer; /* NULL: ones */
  iree_uk_index_t scales_offset;
  void* out_buffer;
  iree_uk_index_t out_offset;
  iree_uk_index_t out_stride0;
  void* workspace_buffer;
  iree_uk_index_t workspace_size; /* bytes */
  iree_uk_index_t M;
  iree_uk_index_t N;
  iree_uk_index_t K;
  iree_uk_index_t rank;
  iree_uk_index_t count;
  int32_t M0;
  int32_t N0;
  int32_t K0;
  uint32_t flags;
} iree_uk_mi355x_adapter_mmt4d_params_t;

/*===--------------------------------------------------------------------===*/
/* Entry points shared with the reference.                                    */
/*===--------------------------------------------------------------------===*/

/* out[M,N,M0,N0] (+)= lhs[M,K,M0,K0] * rhs[N,K,N0,K0]^T.
 * Replaces: mmt4d.h:14-21 (flat form), mmt4d_internal.h:35 (struct form),
 * implemented by mmt4d.c:115-177. `cpu_data` is accepted and ignored (may be
 * NULL). IREE_UK_FLAG_MMT4D_ALLOW_GENERIC_FALLBACK_TILE_FUNCTION is accepted;
 * tile shapes without an MFMA kernel always run on the generic GPU kernel.
 * Strides (the reference checks none, mmt4d.c:12-48): lhs_stride0 and
 * rhs_stride0 may be anything non-negative, 0 and values shorter than a panel
 * included (panels that coincide or overlap are only read). Deviations, both
 * reported through the failure handler with the output left untouched: output
 * rows that overlap (M > 1 and out_stride0 < N * M0 * N0; they are written
 * concurrently here) and negative strides where there is more than one row.
 * Tiles one row tall (M0 = 1) make a row-major [M, K] matrix the lhs and a
 * row-major [M, N * N0] matrix the result as they stand: no pack of the lhs
 * and no unpack are needed then. */
void iree_uk_mmt4d(const void* lhs_buffer, iree_uk_index_t lhs_offset,
                   iree_uk_index_t lhs_stride0, const void* rhs_buffer,
                   iree_uk_index_t rhs_offset, iree_uk_index_t rhs_stride0,
                   void* out_buffer, iree_uk_index_t out_offset,
                   iree_uk_index_t out_stride0, iree_uk_index_t M,
                   iree_uk_index_t N, iree_uk_index_t K, int32_t M0, int32_t N0,
                   int32_t K0, uint32_t flags, const uint64_t* cpu_data);
void iree_uk_mmt4d_p(const iree_uk_mmt4d_params_t* params);

/* Bit 0 is set iff a kernel specialised for (type, M0, N0, K0) exists, here an
 * MFMA or bandwidth-tuned kernel rather than the one-thread-per-element one.
 * Replaces: mmt4d.h:25-27, mmt4d_internal.h:40, mmt4d.c:143-149,179-185. */
uint32_t iree_uk_mmt4d_info(int32_t M0, int32_t N0, int32_t K0, uint32_t flags,
                            const uint64_t* cpu_data);
uint32_t iree_uk_mmt4d_info_p(const iree_uk_mmt4d_params_t* params);

/* 2-D -> 4-D tiled copy with padding and optional inner/outer transposes.
 * Replaces: pack.h:26-34, pack_internal.h:32, pack.c:315-352. */
void iree_uk_pack(const void* in_buffer, iree_uk_index_t in_offset,
                  iree_uk_index_t in_stride0, iree_uk_index_t in_stride1,
                  void* out_buffer, iree_uk_index_t out_offset,
                  iree_uk_index_t out_stride0, iree_uk_index_t out_stride1,
                  iree_uk_index_t in_size0, iree_uk_index_t in_size1,
                  iree_uk_index_t out_size0, iree_uk_index_t out_size1,
                  iree_uk_index_t out_size2, iree_uk_index_t out_size3,
                  uint64_t padding_value, uint32_t flags,
                  const uint64_t* cpu_data);
void iree_uk_pack_p(const iree_uk_pack_params_t* params);

/* Inverse of pack; writes only the out_size0 x out_size1 logical region.
 * Replaces: unpack.h:17-25, unpack_internal.h:31, unpack.c:249-285. */
void iree_uk_unpack(const void* in_buffer, iree_uk_index_t in_offset,
                    iree_uk_index_t in_stride0, iree_uk_index_t in_stride1,
                    void* out_buffer, iree_uk_index_t out_offset,
                    iree_uk_index_t out_stride0, iree_uk_index_t out_stride1,
                    iree_uk_index_t in_size0, iree_uk_index_t in_size1,
                    iree_uk_index_t in_size2, iree_uk_index_t in_size3,
                    iree_uk_index_t out_size0, iree_uk_index_t out_size1,
                    uint32_t flags, const uint64_t* cpu_data);
void iree_uk_unpack_p(const iree_uk_unpack_params_t* params);

/* Tile sizes the matmul kernels of this library prefer for an operand.
 * Replaces: query_tile_sizes.h:29-31, query_tile_sizes.c:34-75. */
void iree_uk_query_tile_sizes_2d(
    const iree_uk_query_tile_sizes_2d_params_t* params,
    iree_uk_query_tile_sizes_2d_out_params_t* out_params);

/* Called when a parameter check or a HIP call fails. The library provides a
 * weak default that prints to stderr and aborts; an embedder may define its
 * own (reference: common.h:307-321 leaves the definition to the embedder). If
 * the handler returns, the entry point returns without launching anything. */
void iree_uk_assert_fail(const char* file, int line, const char* function,
                         const char* condition);

/*===--------------------------------------------------------------------===*/
/* Entry points without a counterpart in the reference.                       */
/*===--------------------------------------------------------------------===*/

/* The in-dispatch int8 microkernel of the ROCm backend's calling convention
 * for gfx950 (iree_amd/csrc/device/iree_uk_amdgpu_multi_mma_mfma_i32_16x16x64_i8.h;
 * the reference has the gfx942 one, compiler/plugins/target/ROCM/builtins/
 * ukernel/iree_uk_amdgpu_multi_mma_mfma_i32_16x16x32_i8.c:82-181), run over a
 * grid of outer_m x outer_n data-tiled tiles, one workgroup each:
 *   a: [outer_m][k_size][subgroups_m][intrinsics_m][64][intrinsics_k] vectors of 16 int8,
 *   b: [outer_n][k_size][subgroups_n][intrinsics_n][64][intrinsics_k],
 *   c: [outer_m][outer_n][subgroups_m][subgroups_n][intrinsics_m][intrinsics_n][64] vectors of 4 int32,
 * c += a * b^T in the MFMA's operand layout (lane l of an A/B vector block: row
 * l % 16, K bytes 16*(l / 16)..+15 of 64; lane l of a C block: rows
 * 4*(l / 16)+{0..3}, column l % 16). Device pointers only. The parameter
 * combinations are compile-time instantiations; returns 0, or a HIP error
 * code (hipErrorInvalidValue for a combination that is not instantiated). It
 * exists to test and measure the device microkernel; there is no host entry
 * point like it in the reference. */
int iree_uk_mi355x_multi_mma_i32_16x16x64_i8(const void* a, const void* b, void* c, long long outer_m,
                                             long long outer_n, int32_t k_size, int32_t intrinsics_m,
                                             int32_t subgroups_m, int32_t intrinsics_n, int32_t subgroups_n,
                                             int32_t intrinsics_k);

/* Quantises a matrix into microscaled tiles: in[in_size0][in_size1] of f32,
 * f16 or bf16, element (i, k) at i * in_stride0 + k * in_stride1, into codes
 * out[out_size0][out_size1][out_size2][out_size3] as iree_uk_pack tiles them
 * and one scale byte for each 32 consecutive values of a tile's row,
 * scales[out_size0][out_size1][out_size2][out_size3 / 32]. out_size3 is a
 * multiple of 32. A 4-bit code with an even index lies in the low half of its
 * byte. Strides in_stride0 = 1, in_stride1 = pitch read a transposed matrix.
 * Tiles one row tall (out_size2 = 1, out_size3 = out_stride0 = the padded
 * row) are the row-major form.
 *   For a block with the largest magnitude a, all finite:
 *     scale byte b = max(floor(log2 a) + 127 - e, 0), e = 2 (E2M1) or 8 (E4M3),
 *     code = the element nearest to x / 2^(b - 127), ties to the even code, the
 *     largest element (6 or 448) beyond it; a = 0 gives b = 0 and zero codes.
 *   A block that holds an infinity or a NaN: scale byte 255 (NaN), zero codes.
 *   What pads the matrix to whole tiles counts as zero.
 * The outputs may not overlap each other, an input or, row for row,
 * themselves. */
void iree_uk_mi355x_mx_pack_p(const iree_uk_mi355x_mx_pack_params_t* params);

/* The inverse: code * 2^(scale - 127), rounded to nearest even in the output's
 * type (infinity beyond its range; scale byte 255 and the NaN codes of E4M3 are
 * NaN). Writes only the out_size0 x out_size1 logical region, element (i, k) at
 * i * out_stride0 + k * out_stride1; rows of the result may not overlap or
 * interleave (out_stride0 > (out_size1 - 1) * out_stride1). */
void iree_uk_mi355x_mx_unpack_p(const iree_uk_mi355x_mx_unpack_params_t* params);

/* iree_uk_mmt4d of microscaled operands: out[M,N,M0,N0] (+)= lhs * rhs^T with
 * lhs[M,K,M0,K0] of E2M1 or E4M3 and rhs[N,K,N0,K0] of E2M1, their scales
 * [M,K,M0,K0/32] and [N,K,N0,K0/32] as iree_uk_mi355x_mx_pack_p writes them.
 * K0 is a multiple of 32. Sums are in f32; the result is rounded once to f16 or
 * bf16 where that is its type (with IREE_UK_MI355X_FLAG_MX_MMT4D_ACCUMULATE the
 * destination's value is added before that rounding). A scale byte of 255 makes
 * every result that its block takes part in NaN, zero codes or not. Products
 * and sums below the smallest normal f32 may come out as zero; where the
 * magnitudes of a result's products add up to 2^128, it may be an infinity or
 * NaN. No bit of a product is lost before it is added, for any type of result.
 * The order of summation is fixed for a call's parameters: the same call gives
 * the same bits.
 * The fast kernels take a K * K0 of whole chunks of 128, operands whose K0 is
 * 128 or whose tiles are one row tall (a row-major matrix with row-major
 * scales), and buffers and strides that are multiples of 16 bytes (scales: of
 * 4); for many rows, lhs tiles whose height is 1 or a multiple of 8. Rhs tiles
 * of 16 x 128 suit them best. Others run on a kernel with one thread for each
 * result. The result may not overlap an operand or, row for row, itself. */
void iree_uk_mi355x_mx_mmt4d_p(const iree_uk_mi355x_mx_mmt4d_params_t* params);

/* Root-mean-square norm of the rows of a matrix, with the residual's addition,
 * into rows that a product reads as its lhs with tiles one row tall. For each
 * of size0 rows of size1 values:
 *   s = in + residual, rounded to their type; stored in `sum` if there is one
 *       (which may be `in` or `residual` itself)
 *   r = 1 / sqrt(mean(s^2) + epsilon), summed in f64, rounded once to f32
 *   y = (s * r) * weight in f32 (weight: the type of `in`, or f32 with
 *       IREE_UK_MI355X_FLAG_RMS_NORM_WEIGHT_F32)
 * and the row of out_size1 >= size1 values, zeros behind the size1 ones, is
 *   S8: q = y * (1 / scale) rounded to nearest even, for iree_uk_mmt4d's S8S8S32
 *       and S8S4S32; scales: one f32 a row, scale = max(max|y| / 127, 2^-126).
 *       A row with a y that is not finite: scale NaN, all q zero.
 *   E4M3, E2M1: codes and scale bytes as iree_uk_mi355x_mx_pack_p makes them of
 *       y, [size0][out_size1 / 32] bytes, rows scales_stride0 apart.
 *       out_size1 is a multiple of 32.
 * `sum` needs a residual. The outputs may not overlap each other or an input,
 * but for a `sum` at exactly the place of `in` or `residual`. */
void iree_uk_mi355x_rms_norm_p(const iree_uk_mi355x_rms_norm_params_t* params);

/* The gated part of a feed-forward block, both products in one kernel:
 *   g = lhs * gate^T,  u = lhs * up^T,  out[M,N,M0,N0] = act(g) * u
 * with lhs[M,K,M0,K0], gate[N,K,N0,K0] and up[N,K,N0,K0] as iree_uk_mmt4d has
 * its operands, of f16 or bf16. Sums, act and its product are in f32; the result
 * is rounded once, to f16 or bf16, where that is its type.
 *   SILU:    act(x) = x * s(x), s(x) = 1 / (1 + e^-x)
 *   GELU:    act(x) = x * s(2 * sqrt(2 / pi) * (x + 0.044715 * x^3)), the tanh form
 *   SIGMOID: act(x) = s(x)
 * x * s(x) is NaN where x is minus infinity.
 *   gate_pre, up_pre: [M,N,M0,N0], of the operands' type or, with PRE_F32, of f32.
 *   With PRE_LOAD what they hold is added to g and u first (adapters, or with a
 *   stride of 0 and tiles one row tall a bias); with PRE_STORE g and u are stored
 *   there, for the backward pass. With both they are updated in place. The
 *   result is computed from g and u as they are ahead of that rounding.
 * The order of summation is fixed for a call's parameters: the same call gives
 * the same bits.
 * The fast kernels take operands with tiles one row tall or a K0 of 8, 16 or 32,
 * and buffers and strides that are multiples of 16 bytes; others run on a kernel
 * with one thread for each result. What is written may not overlap an operand,
 * another result or, row for row, itself. */
void iree_uk_mi355x_gated_mmt4d_p(const iree_uk_mi355x_gated_mmt4d_params_t* params);

/* Its backward pass. From lhs, gate, up, the stored gate_pre (g) and up_pre (u),
 * and out_grad[M,N,M0,N0], the gradient of out:
 *   dg = out_grad * u * act'(g),  du = out_grad * act(g)
 *   lhs_grad[M,K,M0,K0]  = dg * gate + du * up
 *   gate_grad[N,K,N0,K0] (+)= dg^T * lhs,  up_grad[N,K,N0,K0] (+)= du^T * lhs
 * The result's type of the type flag is that of out_grad and of all gradients;
 * with ACCUMULATE the gradients of the weights are added to what they hold. dg
 * and du are rounded to the operands' type in between, which the matrix
 * instructions take, whatever the result's type: each is within 2^-8 (bf16) or
 * 2^-11 (f16) of itself, or in f16 within 2^-39 of the call's largest, which a
 * power of two brings into f16's range first, however large or small they are.
 * The sums over them are in f32 and rounded once. A gradient
 * whose buffer is NULL is not computed, and gate and up are not read without
 * lhs_grad, nor lhs without the gradients of the weights. The same call gives
 * the same bits. The fast kernels ask gate and up, for lhs_grad, and lhs, for the
 * others, to have tiles of 1, 2, 4, .. 32 rows and a multiple of 8 columns (one
 * row tall: of 8 columns in all), and to be aligned as above.
 *   workspace: device memory of iree_uk_mi355x_gated_mmt4d_backward_workspace()
 *   bytes, 256-byte aligned, which is written before it is read and holds
 *   nothing afterwards: dg and du, in f16 what their largest is, and where
 *   lhs_grad has few rows parts of its sums in f32. Calls that may run at the
 *   same time, graphs that hold them included, need workspaces of their own. (In
 *   synchronous mode it may be host memory like any other buffer; it is not
 *   touched then.) */
void iree_uk_mi355x_gated_mmt4d_backward_p(const iree_uk_mi355x_gated_mmt4d_backward_params_t* params);
/* Bytes of workspace for a call with these sizes, flags and gradients (0 where
 * the call would be refused, which is reported as by the call). */
iree_uk_index_t iree_uk_mi355x_gated_mmt4d_backward_workspace(
    const iree_uk_mi355x_gated_mmt4d_backward_params_t* params);

/* Low-rank adapters of many requests at once, beside a product that they share:
 * for each row i of the M * M0 rows of lhs[M,K,M0,K0],
 *   out[i] (+)= scales[a] * (lhs[i] * down[a]^T) * up[a]^T,  a = index[i]
 * with down[count][rank][K * K0] (adapters down_stride0 apart, rows
 * down_stride1), up[count][N * N0][rank] (up_stride0, up_stride1), both of the
 * operands' type and row-major, and scales of f32. A row whose index is
 * negative, or count and more, has no adapter: nothing is added, and without
 * ACCUMULATE its results are zero. With ACCUMULATE out holds the result of
 * iree_uk_mmt4d with the same lhs, M, N, M0, N0; or out is what
 * iree_uk_mi355x_gated_mmt4d_p loads (PRE_LOAD). Products and sums are in f32,
 * rank sums included; the result is rounded once where it is f16 or bf16 (with
 * ACCUMULATE the destination's value is added before that). Rows may come in
 * any order: sixteen at a time share the reads of an adapter, those next to each
 * other or, of many rows and few adapters, wherever they are.
 * The same call gives the same bits, and a row's do not depend on the adapters
 * of other rows. The fast kernels multiply a rank sum by `up` as two or three
 * floats of its type that add up to it (of f16 within 2^-24 of it, or 2^-39 of
 * the row's largest finite one), so that an infinite value of `up` gives
 * infinities or NaN. They take an lhs as above and a `down` whose address and
 * strides are multiples of 16 bytes; `up` may lie anywhere, but takes two to
 * three times as long where it is not aligned like that or rank is no multiple
 * of 8.
 *   workspace: as above, of iree_uk_mi355x_adapter_mmt4d_workspace() bytes; it
 *   holds rank sums in f32 and, where rows are put in order, that. */
void iree_uk_mi355x_adapter_mmt4d_p(const iree_uk_mi355x_adapter_mmt4d_params_t* params);
iree_uk_index_t iree_uk_mi355x_adapter_mmt4d_workspace(const iree_uk_mi355x_adapter_mmt4d_params_t* params);

/* iree_uk_mmt4d_p for callers that cannot allocate. It has no counterpart in
 * the reference (whose microkernels never allocate, being CPU code); it is for
 * callers that may not call hipMalloc where they call a microkernel: tight
 * serving loops, harnesses that forbid allocation, code around HIP graph
 * capture. Same parameters, checks, kernels and results as iree_uk_mmt4d_p.
 * The difference: operands at host addresses are mirrored in a fixed array of
 * IREE_UK_MI355X_NOALLOC_MAX_STAGED_BYTES of device memory that the library's
 * code object holds on every device it runs on until the process ends, instead
 * of in staging buffers grown with hipMalloc. Each host operand takes its span
 * (first to last touched byte) rounded up to 256 bytes; a call whose host
 * operands need more in total reports "host operands exceed ..." through the
 * failure handler and returns without launching. Device operands take none.
 * The call makes no hipMalloc/hipFree. All calls on one device share that
 * array, one at a time: a call with host operands holds it from its first
 * upload until its results are back on the host, and a second such call that
 * arrives on the same device meanwhile (from another thread) is not run: it
 * reports "static staging memory busy" through the failure handler and
 * returns, leaving its output untouched; the caller may repeat it. The array
 * keeps the previous call's bytes, and nothing read from it is ever older
 * than the current call's own uploads. iree_uk_mi355x_init resolves the
 * array's address ahead of the first call.
 * Under stream capture itself only the asynchronous mode can be used (a
 * synchronous call copies and synchronises, which capture forbids), and that
 * mode takes device operands only: nothing is staged there, and this entry
 * point then does exactly what iree_uk_mmt4d_p does, which allocates nothing
 * for device operands either. */
#define IREE_UK_MI355X_NOALLOC_MAX_STAGED_BYTES (16 * 1024 * 1024)
void iree_uk_mi355x_mmt4d_noalloc_p(const iree_uk_mmt4d_params_t* params);

/* Library version, MAJOR*10000 + MINOR*100 + PATCH. */
int iree_uk_mi355x_version(void);

/* Selects the HIP device for the calling thread's launches and checks that it
 * is a gfx950 part; a negative ordinal checks the thread's current device
 * without selecting another. Returns 0 on success, a HIP error code otherwise.
 * Calling it is optional: the first launch uses the current HIP device. */
int iree_uk_mi355x_init(int device_ordinal);

/* Per-thread launch mode.
 *   stream:  a hipStream_t cast to void* (NULL = the HIP null stream).
 *   asynchronous == 0 (default): each entry point returns after its results are
 *     visible, like the CPU microkernels. Operands whose `buffer + offset` is
 *     not a device address are staged: copied to device memory owned by the
 *     library, computed there, and the touched rows copied back.
 *   asynchronous != 0: entry points only enqueue work on `stream` and return;
 *     every operand must be device-accessible; nothing is staged or
 *     synchronised. */
void iree_uk_mi355x_set_stream(void* stream, int asynchronous);

/* Replaces the failure handler for the calling process (NULL restores
 * iree_uk_assert_fail). Meant for hosts that cannot provide a strong
 * iree_uk_assert_fail symbol at link time. */
typedef void (*iree_uk_mi355x_fail_handler_t)(const char* file, int line,
                                              const char* function,
                                              const char* condition);
void iree_uk_mi355x_set_fail_handler(iree_uk_mi355x_fail_handler_t handler);

/* Name of the kernel the calling thread's most recent entry point launched
 * ("" if it returned early). Static storage; do not free. */
const char* iree_uk_mi355x_last_kernel(void);

#ifdef __cplusplus
}
#endif

#endif /* IREE_UK_MI355X_H_ */
