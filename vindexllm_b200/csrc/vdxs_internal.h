// vdxs_internal.h - declarations shared by the C-ABI layer (vdxs_api.cpp) and the
// sm_100a kernels (vdxs_kernels.cu). Not part of the public ABI.
#pragma once

#include <cstdint>
#include <mutex>
#include <string>

#include <cuda_runtime.h>

namespace vdxs {

constexpr int kThreads = 256;        // threads per CTA in every sampling kernel
constexpr int kMaxTopK = 1024;       // largest top_k served by the stream path (larger: the large top-k kernel)
constexpr int kMaxHistory = 8192;    // largest history stride served by the penalty prep
constexpr int kFaithfulSub = 512;    // elements per sub-tile of the min-buffer emulation
constexpr int kFaithfulSlots = 12;  // candidate regions of the min-buffer emulation, in units of kFaithfulSub entries
constexpr int kTauStride = 32;       // words between rows of the stream path's row bounds (one L2 line)

enum Path : int { kGreedy = 0, kTopK = 1, kFull = 2 };

// Unembedding matvec (vdxs_unembed.cu): input rows per launch and their shared memory.
constexpr int kMaxUnembedBatch = 8;
constexpr size_t kUnembedSmemBytes = 200 * 1024;

// Device workspace owned by a context (TVdxSampler.EnsureWorkspace analogue,
// Sampler.pas:250-263). Grown on demand; never shrunk until the context dies.
struct Workspace {
    uint2* cand = nullptr;          // stage-1 (key, index) candidates: [rows * cand_cap] (stream path)
    size_t cand_cap = 0;            // elements
    uint32_t* rhist = nullptr;      // [rows * kRowHistWords] stream path key histograms, self-resetting
    size_t rhist_cap = 0;
    uint32_t* row_cnt = nullptr;    // [rows] stream path list counts, self-resetting
    size_t row_cnt_cap = 0;
    unsigned long long* unit_next = nullptr;  // [2] stream path slot claims and finished warps, self-resetting
    uint32_t* row_counter = nullptr;  // [rows] completion counters, self-resetting
    size_t row_counter_cap = 0;
    uint32_t* row_tau = nullptr;      // [rows * kTauStride] stream path K-th key bounds, self-resetting
    size_t row_tau_cap = 0;
    int32_t* pen_ids = nullptr;     // [rows * pen_stride] sorted unique history ids
    float* pen_vals = nullptr;      // [rows * pen_stride] penalised values
    int32_t* pen_cnt = nullptr;     // [rows]
    uint32_t* pen_bits = nullptr;   // [rows * ceil(vocab / 32)] stream path penalised-id bitmaps, self-resetting
    size_t pen_bits_cap = 0;
    size_t pen_cap = 0;             // rows * pen_stride
    size_t pen_rows_cap = 0;
    uint32_t* fmax = nullptr;       // [rows * nchunks] full path: chunk max keys
    double* fsum = nullptr;         // [rows * nchunks] full path: chunk sums
    size_t full_cap = 0;
    uint2* shard_send = nullptr;    // [rows * K] sharded: local candidates
    uint2* shard_recv = nullptr;    // [ranks * rows * K]
    size_t shard_send_cap = 0, shard_recv_cap = 0;
    uint64_t* lk_buf = nullptr;     // top_k above the stream path's maximum: per-CTA sort buffers and slots
    size_t lk_cap = 0;              // 64-bit words
    float* unembed_logits = nullptr;  // vdxs_sample_unembed_q4_0: [rows * vocab] logits
    size_t unembed_cap = 0;
    int8_t* i8_q = nullptr;           // vdxs_sample_unembed_i8: [rows * pitch] normed hidden states
    float* i8_scale = nullptr;        // and their scales [rows]; its logits are unembed_logits
    size_t i8_q_cap = 0, i8_scale_cap = 0;
    int32_t* err = nullptr;         // device error word (0 = ok)
    // host-buffer entry point staging
    void* d_logits = nullptr;
    size_t d_logits_cap = 0;
    int32_t* d_hist = nullptr;
    size_t d_hist_cap = 0;
    int32_t* d_hcnt = nullptr;
    float* d_unif = nullptr;
    int32_t* d_tok = nullptr;
    size_t d_rows_cap = 0;
    int32_t* h_tok_pinned = nullptr;
};

// Everything one sampling call needs, already validated by the API layer.
struct SampleArgs {
    const void* logits = nullptr;
    int dtype = 0;
    int B = 0;
    int V = 0;                       // local vocab (the shard size when sharded)
    int64_t stride = 0;              // elements between rows
    const int32_t* hist = nullptr;
    int64_t hist_stride = 0;
    const int32_t* hist_count = nullptr;
    const float* uniform = nullptr;
    int32_t* tokens = nullptr;
    uint32_t* flags = nullptr;
    int32_t* out_idx = nullptr;
    float* out_prob = nullptr;
    int out_k = 0;
    // resolved configuration
    int path = kGreedy;
    int K = 1;
    float inv_temp = 1.0f;
    float min_p = 0.0f;
    float top_p = 1.0f;
    float penalty = 1.0f;
    bool penalty_on = false;
    int tie_mode = 0;
    // sharding
    int64_t vocab_offset = 0;
    int64_t vocab_total = 0;
    bool local_emit = false;         // emit local top-K candidates instead of drawing
    cudaStream_t stream = nullptr;
    // diagnostics
    cudaEvent_t ev_begin = nullptr;  // recorded just before the dominant pass
    cudaEvent_t ev_end = nullptr;    // recorded just after it
    int64_t* launches = nullptr;     // incremented per kernel launch
};

struct LaunchPlan {
    int chunk = 0;    // full path: elements per CTA; cluster path: elements per CTA of a row
    int nchunks = 0;  // chunks per row (full-softmax path: CTAs per row)
    int span = 1;     // cluster path: bytes of the staged row chunk
    int nspans = 0;   // stream paths: stage-1 pieces per row
    int elems = 32;   // stream path: warp list registers R (0 = wide stream path)
    bool stream = false;  // top-k path: persistent stream kernel + finish kernel
    bool cluster = false; // top-k path, small batches: one thread-block cluster per row
    bool large = false;   // top-k path, top_k above kMaxTopK: one CTA per row, global workspace
    int large_grid = 0;   // large top-k kernel grid (CTAs)
    size_t large_smem = 0;  // large top-k kernel shared memory
    int cluster_ctas = 8; // CTAs per cluster
    int grid = 0;         // stream kernel grid (CTAs)
    int cand_cap = 0;     // top-k path: candidates each stage-1 list may hold (stream path: per row)
    int gather_cap = 0;   // stream path: finish kernel gather capacity
    long long items = 0;  // top-k path: stage-1 candidate lists
    int slots = 0;        // stream path: 4 KB slots per row
    int unit_slots = 0;   // stream path: slots per claimed unit
    size_t smem = 0;
    size_t smem2 = 0;     // finish kernel shared memory
};

// Host-side launchers (vdxs_kernels.cu). Return cudaSuccess or the launch error;
// `err` receives a message for argument/capacity problems (returned as
// cudaErrorInvalidValue).
cudaError_t plan_topk(const SampleArgs& a, int device_smem_optin, LaunchPlan* plan, std::string* err);
cudaError_t plan_full(const SampleArgs& a, LaunchPlan* plan, std::string* err);
// Makes the error word, cleared, where the context has none yet.
cudaError_t ensure_error_word(Workspace& ws);
cudaError_t ensure_workspace(Workspace& ws, const SampleArgs& a, const LaunchPlan& plan, int ranks,
                             cudaStream_t stream, std::string* err);
cudaError_t launch_sample(const SampleArgs& a, const LaunchPlan& plan, Workspace& ws, std::string* err);
cudaError_t launch_merge_draw(const SampleArgs& a, int ranks, Workspace& ws, std::string* err);
// Unembedding (vdxs_unembed.cu): Q4_0 repack and the matvec in the reference shader's order.
int q4_0_words_per_lane(int in_dim);
size_t q4_0_packed_bytes(int in_dim, int out_dim);
int unembed_chunk_rows(int in_dim);
cudaError_t q4_0_repack(const uint8_t* src, int in_dim, int out_dim, uint32_t* nib, uint16_t* scales,
                        cudaStream_t stream);
cudaError_t q4_0_matvec(const uint32_t* nib, const uint16_t* scales, int in_dim, int out_dim, const float* x,
                        int batch, float* out, cudaStream_t stream, int* launches);
// Norm, residual and 8-bit output, and the 8-bit unembedding (vdxs_i8.cu, vdxs_i8_product.cu).
struct NormI8Args {
    const void* x = nullptr;
    int64_t x_stride = 0;
    const void* residual = nullptr;
    int64_t residual_stride = 0;
    int dtype = 0;
    const void* weight = nullptr;
    int weight_dtype = 0;
    int rows = 0, dim = 0;
    float eps = 0.0f;
    void* hidden = nullptr;
    int64_t hidden_stride = 0;
    int8_t* q = nullptr;
    int64_t q_stride = 0;
    float* scale = nullptr;
};
struct I8Matrix {            // weights as the product reads them
    int8_t* q = nullptr;     // [out_dim][pitch], the bytes behind in_dim are not read
    float* scale = nullptr;  // [out_dim]
    int in_dim = 0, out_dim = 0;
    int64_t pitch = 0;       // bytes between rows: in_dim rounded up to 16
    alignas(64) unsigned char map[128] = {};  // tensor map of q (map_weights_i8)
};
// Makes w.map, once the other members are set.
cudaError_t map_weights_i8(I8Matrix& w);
// cudaFuncAttributeMaxDynamicSharedMemorySize of a kernel on each device. It belongs to the process,
// and contexts on other threads raise it too: check, call and note are one step, and it is
// never lowered.
struct SmemLimit {
    std::mutex mu;
    int have[64] = {};
    template <typename F>
    cudaError_t raise(F* kernel, size_t bytes) {
        if (bytes <= 48 * 1024) return cudaSuccess;
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return e;
        if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
        std::lock_guard<std::mutex> lock(mu);
        if (have[dev] >= (int)bytes) return cudaSuccess;
        e = cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
        if (e == cudaSuccess) have[dev] = (int)bytes;
        return e;
    }
};
cudaError_t rms_norm_i8(const NormI8Args& a, int sm_count, cudaStream_t stream);
// Rows of fp32/bf16/fp16 (format 0..2) or Q4_0 blocks (4) to 8 bits with a scale per row.
cudaError_t quantise_rows_i8(const void* src, int format, int64_t row_stride, const I8Matrix& w, cudaStream_t stream);
// The product's form for its sizes.
constexpr int kI8TileM = 128;   // vocabulary entries of a tile
constexpr int kI8ChunkK = 128;  // bytes of a row in a stage: one swizzle span
constexpr int kI8MaxN = 256;    // batch columns of a tile
struct I8ProductForm {
    enum Mode : int { kSingle = 0, kPair = 1, kSplit = 2 };
    int mode = kSingle, split = 1, n_tiles = 1, n = 16;
};
inline I8ProductForm i8_product_form(int batch, int in_dim, int out_dim, int sm_count) {
    I8ProductForm f;
    // Equal column tiles of at most 256, a multiple of 16 wide (of 32 in pairs).
    f.n_tiles = (batch + kI8MaxN - 1) / kI8MaxN;
    const int64_t tiles = (int64_t)((out_dim + kI8TileM - 1) / kI8TileM) * f.n_tiles;
    const int chunks = (in_dim + kI8ChunkK - 1) / kI8ChunkK;
    // Pairs where the batch operand weighs, the sums are long and every SM has a tile: batch 512 of
    // 262144 x 2560 291 us against 312, batch 256 of 32003 x 3840 35.3 against 38.5; but batch 256
    // of 262144 x 1152 109 against 101, and batch 512 of 8000 x 4096 18.9 against 17.2.
    const bool pair = batch > 128 && in_dim >= 2048 && tiles > sm_count;
    // A split's share is four chunks at least, and its clusters fit the GPU at once (8-CTA clusters
    // fill only part of a GPU's SM groups). Batch 1 of 1000 x 8192 7.9 us with 8 parts against
    // 22.2 with one, of 8000 x 4096 9.4 with 2 against 12.8.
    for (int s = 2; s <= 8 && tiles * s <= sm_count * (s < 8 ? 7 : 6) / 8 && chunks >= 4 * s; s *= 2) f.split = s;
    f.mode = pair ? I8ProductForm::kPair : f.split > 1 ? I8ProductForm::kSplit : I8ProductForm::kSingle;
    const int step = pair ? 32 : 16, columns = (batch + f.n_tiles - 1) / f.n_tiles;
    f.n = (columns + step - 1) / step * step;
    return f;
}
cudaError_t unembed_i8(const I8Matrix& w, const int8_t* q, int64_t q_stride, const float* scale, int batch,
                       void* logits, int dtype, int64_t logits_stride, int32_t* err, int sm_count, cudaStream_t stream,
                       int* launches);
// Beam search (vdxs_beam.cu).
struct BeamWorkspace {
    unsigned long long* cand = nullptr;  // [rows][chunks][beams] each chunk's best (key, token), best first
    double* part = nullptr;              // [rows][chunks][2] each chunk's maximum and sum of exponentials
    unsigned long long* best = nullptr;  // [rows][beams] each row's best
    double* lse = nullptr;               // [rows] log of the sum of exponentials
    uint32_t* row_done = nullptr;        // [rows] chunks done, self-resetting
    uint32_t* prompt_done = nullptr;     // [batch] rows done, self-resetting
    int32_t* push = nullptr;             // [rows] 1: the row's ring takes the new token
};
struct BeamArgs {
    const void* logits = nullptr;
    int dtype = 0;
    int64_t stride = 0;
    int batch = 0, beams = 0, vocab = 0, chunks = 0, chunk = 0;
    float penalty = 1.0f;
    int window = 0;
    double alpha = 0.0;
    int32_t pad = 0;
    const float* scores_in = nullptr;
    const int32_t *lengths_in = nullptr, *finished_in = nullptr, *hist_in = nullptr, *pos_in = nullptr,
                  *count_in = nullptr;
    float* scores = nullptr;
    int32_t *lengths = nullptr, *finished = nullptr, *hist = nullptr, *pos = nullptr, *count = nullptr;
    const int32_t* stop_ids = nullptr;
    int n_stop = 0;
    int32_t *tokens = nullptr, *parents = nullptr;
    bool merge_rows = false;  // set by beam_select: each row's chunks are merged before the prompt
    bool move_rings = false;  // the selection moves the rings itself
    BeamWorkspace ws;
};
// Rings up to this length are moved by the selection where a step has no caches to move.
constexpr int kBeamShortWindow = 1024;
struct BeamCacheArgs {  // vdxs_beam_cache
    const unsigned char* src = nullptr;
    unsigned char* dst = nullptr;
    int64_t src_row = 0, src_segment = 0, dst_row = 0, dst_segment = 0, segment_bytes = 0, segments = 0;
};
// Chunks of a row of `vocab` logits (at most kBeamMaxChunks) and their length.
constexpr int kBeamMaxChunks = 64;
constexpr int kBeamMaxVocab = 8000000;  // kBeamMaxChunks chunks of the longest kind
void beam_plan(int rows, int vocab, int sm_count, int* chunks, int* chunk);
cudaError_t beam_select(const BeamArgs& a, cudaStream_t stream);
// Caches by a.parents; behind a beam_select on the same stream also the rings that it left.
cudaError_t beam_reorder(const BeamArgs& a, bool behind_select, const BeamCacheArgs* caches, int n_caches,
                         cudaStream_t stream, int* launches);
// Device-resident decode state (one thread per row).
cudaError_t launch_device_uniforms(uint64_t* prng, int batch, float* out, cudaStream_t stream);
cudaError_t launch_history_push(int32_t* hist, int32_t* pos, int32_t* count, int window, const int32_t* tokens,
                                int batch, const int32_t* stop_ids, int n_stop, int32_t* stopped,
                                cudaStream_t stream);
void free_workspace(Workspace& ws);
// Clears the device error word and the self-resetting counters (after a failed launch).
cudaError_t reset_device_state(Workspace& ws, cudaStream_t stream);

// Fixed device scratch used by vdxs_sample_noalloc (no allocation on any call).
constexpr size_t kNoAllocScratchBytes = (size_t)32 << 20;
// Byte offset of the device error word inside that array (the first field carved).
constexpr size_t kNoAllocErrOffset = 0;
// Device address of the scratch on the current device (resolved once per device) and
// that device's opt-in shared-memory limit.
cudaError_t noalloc_scratch(void** ptr, int* smem_optin);
// Lays out the workspace of one call inside [base, base + cap) without allocating.
// Returns the bytes the call needs; the pointers are set only when it fits.
size_t carve_workspace(Workspace& ws, unsigned char* base, size_t cap, const SampleArgs& a, const LaunchPlan& plan);

}  // namespace vdxs
