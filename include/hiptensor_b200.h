/* Flat C ABI of libhiptensor_b200.so.
 *
 * The reference library (ROCm/hipTensor 1.4.0) exposes its API with C++ linkage and
 * std::vector-bearing structs, which no FFI can bind. Each function below is the
 * extern "C" twin of one of those entry points: plain pointers, sizes and integers,
 * descriptors behind opaque handles that the library allocates and frees. Argument
 * meaning, status codes and error behaviour are those of the C++ function named in
 * the comment (file:line inside the reference project).
 *
 * Data pointers (A, B, C, D, workspace) are device pointers; alpha/beta are host
 * pointers; all work is enqueued on `stream` (a cudaStream_t passed as void*).
 * Status codes: the hiptensorStatus_t values (0 success, 1 not initialised,
 * 7 invalid value, 8 arch mismatch, 13 execution failed, 14 internal error,
 * 15 not supported, 18 CUDA error, 19 insufficient workspace).
 */
#ifndef HIPTENSOR_B200_H
#define HIPTENSOR_B200_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct htHandle           htHandle;           /* hiptensorHandle_t */
typedef struct htTensorDescriptor htTensorDescriptor; /* hiptensorTensorDescriptor_t */
typedef struct htContractionDesc  htContractionDesc;  /* hiptensorContractionDescriptor_t */
typedef struct htContractionFind  htContractionFind;  /* hiptensorContractionFind_t */
typedef struct htContractionPlan  htContractionPlan;  /* hiptensorContractionPlan_t */
typedef struct htScaledContractionPlan htScaledContractionPlan; /* no counterpart in the reference */
typedef struct htCrossEntropyPlan      htCrossEntropyPlan;      /* no counterpart in the reference */

/* library/include/hiptensor/hiptensor.hpp:41,46 (library/src/hiptensor.cpp:35-104) */
int htCreate(htHandle** handle);
int htDestroy(htHandle* handle);

/* hiptensor.hpp:71 (hiptensor.cpp:216-254) */
const char* htGetErrorString(int status);

/* hiptensor.hpp:60-66 (hiptensor.cpp:106-214). strides == NULL: packed, LAST mode fastest.
 * dataType: 0 f32, 1 f64, 2 f16, 14 bf16, 4 cf32, 5 cf64, and for the block-scaled operations 28 e4m3, 29 e5m2.
 * unaryOp: 1 identity, 2 "sqrt" (= square). */
int htCreateTensorDescriptor(const htHandle* handle, htTensorDescriptor** desc, uint32_t numModes,
                             const int64_t* lens, const int64_t* strides, int dataType, int unaryOp);
int htDestroyTensorDescriptor(htTensorDescriptor* desc);

/* hiptensor.hpp:108-111 (hiptensor.cpp:256-321) */
int htGetAlignmentRequirement(const htHandle* handle, const void* ptr, const htTensorDescriptor* desc,
                              uint32_t* alignmentRequirement);

/* hiptensor.hpp:89-98 (library/src/permutation/hiptensor_permutation.cpp:43-279).
 * typeScalar: 0 f32, 2 f16 (type alpha points to). */
int htPermutation(const htHandle* handle, const void* alpha, const void* A, const htTensorDescriptor* descA,
                  const int32_t* modeA, void* B, const htTensorDescriptor* descB, const int32_t* modeB,
                  int typeScalar, void* stream);

/* hiptensor.hpp:131-145 (library/src/contraction/hiptensor_contraction.cpp:71-219).
 * descC == NULL selects the scale form D = alpha*A*B.
 * typeCompute: 1 f16, 4 f32, 16 f64, 1024 bf16 (hiptensorComputeType_t). */
int htCreateContractionDescriptor(const htHandle* handle, htContractionDesc** desc,
                                  const htTensorDescriptor* descA, const int32_t* modeA, uint32_t alignA,
                                  const htTensorDescriptor* descB, const int32_t* modeB, uint32_t alignB,
                                  const htTensorDescriptor* descC, const int32_t* modeC, uint32_t alignC,
                                  const htTensorDescriptor* descD, const int32_t* modeD, uint32_t alignD,
                                  int typeCompute);
int htDestroyContractionDescriptor(htContractionDesc* desc);

/* hiptensor.hpp:157-159 (hiptensor_contraction.cpp:221-316). algo: -1 default, -6 patient, -8 actor-critic. */
int htCreateContractionFind(const htHandle* handle, htContractionFind** find, int algo);
int htDestroyContractionFind(htContractionFind* find);

/* hiptensor.hpp:170-174 (hiptensor_contraction.cpp:318-419). pref: 1 min, 2 recommended, 3 max. */
int htContractionGetWorkspaceSize(const htHandle* handle, const htContractionDesc* desc,
                                  const htContractionFind* find, int pref, uint64_t* workspaceSize);

/* hiptensor.hpp:191-195 (hiptensor_contraction.cpp:421-604) */
int htCreateContractionPlan(const htHandle* handle, htContractionPlan** plan, const htContractionDesc* desc,
                            const htContractionFind* find, uint64_t workspaceSize);
int htDestroyContractionPlan(htContractionPlan* plan);

/* hiptensor.hpp:218-228 (hiptensor_contraction.cpp:606-855). alpha/beta typed by the compute type. */
int htContraction(const htHandle* handle, const htContractionPlan* plan, const void* alpha, const void* A,
                  const void* B, const void* beta, const void* C, void* D, void* workspace,
                  uint64_t workspaceSize, void* stream);

/* hiptensor.hpp:255-271 (library/src/reduction/hiptensor_reduction.cpp:174-381).
 * opReduce: 3 add, 5 mul, 6 max, 7 min. */
int htReduction(const htHandle* handle, const void* alpha, const void* A, const htTensorDescriptor* descA,
                const int32_t* modeA, const void* beta, const void* C, const htTensorDescriptor* descC,
                const int32_t* modeC, void* D, const htTensorDescriptor* descD, const int32_t* modeD,
                int opReduce, int typeCompute, void* workspace, uint64_t workspaceSize, void* stream);

/* hiptensor.hpp:290-302 (hiptensor_reduction.cpp:383-399) */
int htReductionGetWorkspaceSize(const htHandle* handle, const void* A, const htTensorDescriptor* descA,
                                const int32_t* modeA, const void* C, const htTensorDescriptor* descC,
                                const int32_t* modeC, const void* D, const htTensorDescriptor* descD,
                                const int32_t* modeD, int opReduce, int typeCompute, uint64_t* workspaceSize);

/* No counterpart in the reference. hiptensorReduction for callers that are not allowed to allocate
 * device memory while they work: a plug-in inside a host application that has claimed the whole device
 * heap, a latency-critical loop where cudaMalloc's implicit device synchronisation is not acceptable, a
 * service whose policy forbids device allocations once start-up is over. The scratch of the two-pass reduction (few outputs, long reduced
 * range) is a fixed 8 KiB array inside the library, present on every device that loads the library until
 * the process ends; the call makes no cudaMalloc / cudaFree and uses no caller workspace. Inputs and
 * outputs are still the caller's. Limits and rules:
 *  - a reduction of long contiguous rows whose two-pass scratch would exceed 8 KiB returns 19
 *    (INSUFFICIENT_WORKSPACE) and does nothing; use htReduction with a workspace for it (on B200 this only
 *    concerns fp64 reductions with several hundred outputs). Reductions of short rows or with a contiguous kept
 *    mode use as many slices as the 8 KiB hold, or a single pass;
 *  - the first call on a device looks up the array's device address; make that first call outside any
 *    stream capture;
 *  - all calls on one device share the array, and it keeps the last call's contents. Nothing in it needs
 *    clearing (the first pass overwrites every slot the second pass reads), but two such calls that run
 *    at the same time on one device (different streams) race on it: keep them on one stream or order
 *    them with events. */
int htReductionNoAlloc(const htHandle* handle, const void* alpha, const void* A, const htTensorDescriptor* descA,
                       const int32_t* modeA, const void* beta, const void* C, const htTensorDescriptor* descC,
                       const int32_t* modeC, void* D, const htTensorDescriptor* descD, const int32_t* modeD,
                       int opReduce, int typeCompute, void* stream);

/* No counterpart in the reference, whose handle is bound to one device (hiptensor_contraction.cpp:263-277).
 * Finishes a reduction whose REDUCED mode is split over several devices: every device calls htReduction on
 * its share of A with alpha = 1 and beta = 0, the partial results (laid out like D) are combined by one
 * all-reduce that uses the reduction's operator (sum, product, min, max), and this call then writes
 * D = alpha * partial + beta * C once, in the order of the single-device epilogue
 * (library/src/reduction/reduction_cpu_reference_impl.hpp:45-64). partial, C and D share descD; C may be
 * NULL (beta is then ignored) and partial may alias D. */
int htReductionFinish(const htHandle* handle, const void* alpha, const void* partial, const void* beta, const void* C,
                      void* D, const htTensorDescriptor* descD, int typeCompute, void* stream);

/* ---- 8-bit tensors with a scale for each block of 128 (no counterpart in the reference) ----
 *
 * htBlockQuantize writes A[modeA] (f32, f16, bf16) as Q[modeQ] (e4m3 or e5m2; the modes of A in any order) and f32
 * scales S, so that Q * S is A again up to the 8-bit rounding. blockA gives 1 or 128 for each mode of A; one or two modes
 * of extent above 1 may have 128. S has A's modes in A's order with extents ceil(extent / block). For every block
 *     a = max(max |A|, 2^-100),  S = a / q,  Q = A * (q / a) rounded once to the nearest 8-bit number, ties to even,
 * with q = 448 (e4m3) or 57344 (e5m2); S and q / a are f32 numbers. A block with a NaN gets the scale NaN, one with an
 * infinity the scale infinity: multiplied out, all of either is NaN. Strides of A, Q and S are the caller's (an output
 * needs a place for every element); the modes of block 1 must fold into one (two blocked modes) or two modes. What lies
 * between the rows of Q and S (padding) stays as it was. A contiguous mode and rows at multiples of 16 bytes run fastest.
 *
 * Returns 15 for types, operators and mode groups outside this, 7 for extents that do not fit together. */
int htBlockQuantize(const htHandle* handle, const void* A, const htTensorDescriptor* descA, const int32_t* modeA,
                    const uint32_t* blockA, void* Q, const htTensorDescriptor* descQ, const int32_t* modeQ, float* S,
                    const htTensorDescriptor* descS, void* stream);

/* D[modeD] = alpha * sum over the contracted mode of (A * scaleA) (B * scaleB), + beta * C. A and B are e4m3 or e5m2 (each
 * its own), D is f32, f16 or bf16, C (descC == NULL: none) is described as D is. descScaleA / blockA and descScaleB /
 * blockB are those of htBlockQuantize for A's and B's modes. One mode is contracted, with block 128 in both operands; the
 * free modes of an operand fold into one mode, of block 1 or 128. Each block's products are summed in f32, multiplied by the
 * product of the two scales (an f32 number, which has to be in range), and summed in f32 over the blocks.
 * typeCompute: 4 (f32); alpha and beta point to floats. A mode in A, B and D is not supported (15), as in htContraction. No
 * workspace is needed, and a plan may be used by several calls and streams at once. Operands that are contiguous along the
 * contracted mode, with rows at multiples of 16 bytes, run on the tensor cores; any other strides on FMA. */
int htCreateScaledContractionPlan(const htHandle* handle, htScaledContractionPlan** plan, const htTensorDescriptor* descA,
                                  const int32_t* modeA, const htTensorDescriptor* descScaleA, const uint32_t* blockA,
                                  const htTensorDescriptor* descB, const int32_t* modeB, const htTensorDescriptor* descScaleB,
                                  const uint32_t* blockB, const htTensorDescriptor* descC, const htTensorDescriptor* descD,
                                  const int32_t* modeD, int typeCompute);
int htDestroyScaledContractionPlan(htScaledContractionPlan* plan);
int htScaledContraction(const htHandle* handle, const htScaledContractionPlan* plan, const void* alpha, const void* A,
                        const float* scaleA, const void* B, const float* scaleB, const void* beta, const void* C, void* D,
                        void* stream);

/* ---- softmax cross entropy of a linear head (no counterpart in the reference) ----
 *
 * Logits z = alpha * (H contracted with W) are never kept: they are made, used and dropped piece by piece of the
 * vocabulary. The modes that H and W share are contracted, H's other modes are the tokens (numbered in modeH's order, the
 * last one fastest), W's other modes the classes (numbered likewise). H and W are f16, bf16 or f32, both the same; they and
 * dH and dW start at multiples of 16 bytes; targets are int64, loss, lse and gradLoss f32, one packed value for each token.
 *     lse = log sum over classes of exp z,   loss = lse - z[target];   loss = 0 where target == ignoreIndex
 *     P = (exp(z - lse) - [class == target]) * gradLoss * alpha, 0 where target == ignoreIndex
 *     dH = P contracted with W (laid out like H),   dW = P contracted with H (laid out like W)
 * htCrossEntropyGradient takes lse as htCrossEntropy wrote it; dH or dW may be NULL (not wanted). Rows of H whose target is
 * ignored take no part in the gradient, whatever they hold, and their rows of dH are 0, whatever W holds. A target that is neither a class nor ignoreIndex reads
 * nothing out of range: its loss is NaN, its row of P zero, and the next call on the handle returns 13
 * (EXECUTION_FAILED) once. Sums are f32, softmax statistics too. Of a few tokens P stays f32; else it is rounded to the type of H
 * (f16: scaled by a power of two for the largest finite |gradLoss * alpha| of the tokens that count) but for the targets' entries,
 * which outweigh the others: what rounding takes from them is added in f32 (dW: of at least 16 of a class's tokens). For dW of
 * up to 64 tokens P is a sum of two such numbers. f32 tensors of more than a few tokens are multiplied as sums of three bf16
 * numbers, which is f32's own accuracy; an infinity among them makes NaN of the logits it takes part in.
 *
 * Fastest are H and W contiguous along the contracted mode, in rows at multiples of 16 bytes; W contiguous along the classes takes
 * two to three and a half times as long. dH and dW need a place for every element, and neither they nor the workspace overlap an operand.
 *
 * The workspace holds the pieces: any size from htCrossEntropyGetWorkspaceSize's MIN on (19 below it); with more, pieces
 * are larger and fewer. gradient: 0 for htCrossEntropy, 1 for htCrossEntropyGradient. Two calls that run at the same time (two
 * streams, two captured graphs) need a workspace each. Results do not depend on other calls and are the same every time
 * for the same workspace size. */
int htCreateCrossEntropyPlan(const htHandle* handle, htCrossEntropyPlan** plan, const htTensorDescriptor* descH,
                             const int32_t* modeH, const htTensorDescriptor* descW, const int32_t* modeW, int64_t ignoreIndex,
                             int typeCompute);
int htDestroyCrossEntropyPlan(htCrossEntropyPlan* plan);
int htCrossEntropyGetWorkspaceSize(const htHandle* handle, const htCrossEntropyPlan* plan, int gradient, int pref,
                                   uint64_t* workspaceSize);
int htCrossEntropy(const htHandle* handle, const htCrossEntropyPlan* plan, const void* alpha, const void* H, const void* W,
                   const int64_t* targets, float* loss, float* lse, void* workspace, uint64_t workspaceSize, void* stream);
int htCrossEntropyGradient(const htHandle* handle, const htCrossEntropyPlan* plan, const void* alpha, const void* H,
                           const void* W, const int64_t* targets, const float* lse, const float* gradLoss, void* dH, void* dW,
                           void* workspace, uint64_t workspaceSize, void* stream);

/* hiptensor.hpp:308-338 (library/src/logger.cpp). mask: OR of 1 error, 2 perf, 4 hint, 8 heuristics, 16 api. */
int htLoggerSetMask(int32_t mask);
int htLoggerOpenFile(const char* logFile);

/* Introspection of the host-side planner (no device work; usable without a GPU).
 * Each writes a short human-readable description of the plan the library would run
 * (folded extents, kernel family, tile shape) into buf and returns a status code.
 * They replace nothing in the reference: its selection is CK instance enumeration
 * (library/src/contraction/contraction_selection.cpp:44-195,1687-2214). */
int htDescribePermutationPlan(uint32_t numModes, const int64_t* lensA, const int32_t* modeA, const int32_t* modeB,
                              int dataTypeA, int dataTypeB, char* buf, uint64_t bufSize);
int htDescribeReductionPlan(uint32_t numModesA, const int64_t* lensA, const int64_t* stridesA,
                            const int32_t* modeA, uint32_t numModesD, const int64_t* lensD,
                            const int64_t* stridesD, const int32_t* modeD, int dataType, char* buf,
                            uint64_t bufSize);
int htDescribeContractionPlan(uint32_t numModesA, const int64_t* lensA, const int64_t* stridesA,
                              const int32_t* modeA, int dataTypeA, uint32_t numModesB, const int64_t* lensB,
                              const int64_t* stridesB, const int32_t* modeB, int dataTypeB, uint32_t numModesD,
                              const int64_t* lensD, const int64_t* stridesD, const int32_t* modeD, int dataTypeD,
                              int hasC, int typeCompute, char* buf, uint64_t bufSize);

/* Name of the kernel family the last call on this thread launched ("" if none).
 * For tests and the bench, to show which CUDA path ran. */
const char* htLastKernelName(void);
/* Device status word of the handle: 0, or the code a kernel left when one of its bounded device-side waits ran
 * out (1 permutation, 2 single-CTA f16 kernel, 3 CTA-pair f16 kernel, 4 fp32 tensor-core kernel, 5 block-scaled 8-bit
 * kernel, 6 cross-entropy kernel), or 7 when a cross entropy met a target outside the vocabulary. Reading does not
 * clear it; the next operation on the handle reports HIPTENSOR_STATUS_EXECUTION_FAILED once and clears it. No
 * reference counterpart: the reference's kernels have no device-side waits. */
int htGetDeviceStatus(const htHandle* handle, int32_t* status);
/* The CUDA device that the handle is bound to (the current one when it was made). No reference counterpart. */
int htGetDevice(const htHandle* handle, int32_t* device);
/* Test aid (host-side fault injection): writes the status word as a timed-out kernel would, so that the error
 * path of the next operation can be exercised without making a kernel wait. */
int htInjectDeviceStatus(const htHandle* handle, int32_t code);
/* The library reads its variant switches (environment variables HTB_*, which choose between shipped kernel
 * variants and never change a result beyond the order of summation) once when it is loaded; this reads them
 * again. For tests that set a switch after loading the library. */
void htReloadSwitches(void);
/* Number of kernel launches made by this library since load (all threads). */
uint64_t htKernelLaunchCount(void);

#ifdef __cplusplus
}
#endif
#endif /* HIPTENSOR_B200_H */
