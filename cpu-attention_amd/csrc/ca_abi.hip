// The extern "C" entries declared in include/cpu_attention_hip.h.  Each one checks
// what its kernels assume (the static half of the reference's native validation,
// cpu_attention/_mojo/src/_C.mojo:104-160, 190-205, 249-267, plus the 16-byte
// alignment the vector loads need) and returns CA_DECLINED without launching
// anything otherwise.
#include <stdio.h>

#include <atomic>

#include "ca_device.h"
#include "ca_internal.h"

using namespace ca;

namespace {

bool head_dim_ok(int64_t e) { return e == 32 || e == 64 || e == 128; }
bool dtype_ok(int32_t dt) { return dt == CA_F32 || dt == CA_BF16; }
int64_t esize(int32_t dt) { return dt == CA_BF16 ? 2 : 4; }
bool aligned16(const void* ptr) { return ((uintptr_t)ptr & 15) == 0; }
// An element stride whose byte size keeps 16-byte alignment.
bool stride16(int64_t stride, int32_t dt) { return (stride * esize(dt)) % 16 == 0; }
bool page_ok(int64_t page) { return page > 0 && page % 16 == 0; }

}  // namespace

extern "C" int ca_abi_version(void) { return CA_ABI_VERSION; }

extern "C" const char* ca_version(void) {
  return "cpu-attention gfx950 (MI355X) HIP kernels, ABI " "3";
}

extern "C" const char* ca_status_string(int status) {
  if (status == CA_OK) return "ok";
  if (status == CA_DECLINED) return "declined: arguments outside what the kernels take";
  if (status == CA_SCRATCH_EXCEEDED)
    return "ca_decode_noalloc: the call needs more split-K scratch than the fixed 32 MiB buffer "
           "(a page table of this capacity needs ca_decode with a caller workspace)";
  if (status < 0) return hipGetErrorString((hipError_t)(CA_HIP_ERROR - status));
  return "unknown status";
}

extern "C" int ca_store(const ca_store_args* a, void* stream) {
  if (!a || !dtype_ok(a->dtype) || !head_dim_ok(a->head_dim) || !page_ok(a->page_size))
    return CA_DECLINED;
  if (a->num_tokens < 0 || a->num_heads <= 0 || a->num_blocks < 0) return CA_DECLINED;
  if (a->num_tokens == 0) return CA_OK;
  if (!a->key || !a->value || !a->k_cache || !a->v_cache || !a->slot_mapping) return CA_DECLINED;
  if (!aligned16(a->key) || !aligned16(a->value) || !aligned16(a->k_cache) || !aligned16(a->v_cache))
    return CA_DECLINED;
  // One token is never stepped over, so its stride is not read (a [1, H, E]
  // view may carry any stride there, 0 included).
  const bool one = a->num_tokens == 1;
  if (!one && (!stride16(a->token_stride, a->dtype) || a->token_stride < a->num_heads * a->head_dim))
    return CA_DECLINED;
  const int64_t words = a->head_dim * esize(a->dtype) / 4;
  StoreParams p{};
  p.key = static_cast<const uint32_t*>(a->key);
  p.value = static_cast<const uint32_t*>(a->value);
  p.tok_stride_w = one ? 0 : a->token_stride * esize(a->dtype) / 4;
  p.kc = static_cast<uint32_t*>(a->k_cache);
  p.vc = static_cast<uint32_t*>(a->v_cache);
  p.slots = a->slot_mapping;
  p.ntok = a->num_tokens;
  p.per_seq = 1;
  p.heads = a->num_heads;
  p.page = a->page_size;
  p.nblocks = a->num_blocks;
  return store_launch(p, (int)words, static_cast<hipStream_t>(stream));
}

// Workspace layout: fp32 partial accumulators [slots, E], then (max, sum) pairs
// [slots, 2], one slot per (row, block of 8 tiles of the page table's capacity);
// for calls of kMergeMinRows to kMergeMaxRows rows of at most kMergeMaxBlocks
// blocks, then one 8-byte counter per row (the in-kernel merge).
static int64_t decode_acc_bytes(int64_t slots, int64_t head_dim) {
  return ((slots * head_dim * 4 + 255) / 256) * 256;
}

// slots = rows x blocks per row (0: every row fits one block).
static bool decode_merges(int64_t rows, int64_t slots) {
  return slots > 0 && rows >= kMergeMinRows && rows <= kMergeMaxRows && slots <= rows * kMergeMaxBlocks;
}

static int64_t decode_ws_bytes(int64_t rows, int64_t head_dim, int64_t page, int64_t width, int tile_keys) {
  const int64_t slots = decode_workspace_slots(rows, decode_tiles(width, page, tile_keys));
  return decode_acc_bytes(slots, head_dim) + slots * 2 * 4 + (decode_merges(rows, slots) ? rows * 8 : 0);
}

// The in-kernel merge's per-call tag: n * 0x9E3779B9 for the process's n-th call
// (an odd multiplier, so no tag repeats within 2^32 calls), skipping values
// within 2^24 of zero: never 0 (the value a counter holds between calls), nor the
// small integers of either sign that a reused workspace tends to hold in a
// counter's high word.
static uint32_t next_merge_tag() {
  static std::atomic<uint32_t> n{0};
  constexpr uint32_t kNear = 1u << 24;
  uint32_t t = 0;
  while (t < kNear || t > ~kNear) t = ++n * 0x9E3779B9u;
  return t;
}

extern "C" int64_t ca_decode_workspace_bytes(int64_t num_seqs, int64_t num_heads,
                                             int64_t head_dim, int64_t page_size,
                                             int64_t page_table_width) {
  if (num_seqs < 0 || num_heads < 0 || page_size <= 0 || page_table_width < 0) return -1;
  // The tile size depends on the element size, which the query does not name: it
  // answers for the larger of the bf16 and the fp32 call.
  const int64_t rows = num_seqs * num_heads;
  int64_t most = 0;
  for (int esize : {2, 4}) {
    const int64_t b = decode_ws_bytes(rows, head_dim, page_size, page_table_width,
                                      decode_tile_keys(rows, page_table_width, page_size, head_dim, esize));
    most = b > most ? b : most;
  }
  return most;
}

// ca_decode and ca_decode_noalloc.  The split-K scratch is the caller's workspace,
// or for noalloc the library's fixed buffer.  A call whose partials with the
// preferred tile size do not fit the scratch it has takes 256-key tiles (fewer
// partials per row) if those fit.  With one tile size the need grows with the
// rows, so a workspace sized by ca_decode_workspace_bytes for the largest batch
// holds every smaller batch of the same page table, whichever tile size the
// smaller batch would prefer.
static int decode_entry(const ca_decode_args* a, void* stream, bool noalloc) {
  if (!a || !dtype_ok(a->dtype) || !head_dim_ok(a->head_dim) || !page_ok(a->page_size))
    return CA_DECLINED;
  if (a->num_seqs < 0 || a->num_heads <= 0 || a->num_blocks < 0 || a->page_table_width < 0)
    return CA_DECLINED;
  if (a->num_seqs == 0) return CA_OK;
  // The tile size and the split-K scratch it needs depend on the shapes only; the
  // no-allocation entry refuses a call its buffer cannot hold before anything else.
  const int64_t rows = a->num_seqs * a->num_heads;
  const int64_t have = noalloc ? CA_DECODE_NOALLOC_SCRATCH_BYTES
                               : (a->workspace && aligned16(a->workspace) && a->workspace_bytes > 0
                                      ? a->workspace_bytes : 0);
  int tile_keys = decode_tile_keys(rows, a->page_table_width, a->page_size, a->head_dim, a->dtype == CA_BF16 ? 2 : 4);
  int64_t need = decode_ws_bytes(rows, a->head_dim, a->page_size, a->page_table_width, tile_keys);
  if (need > have && tile_keys != kDecodeLongTile) {
    const int64_t need_long = decode_ws_bytes(rows, a->head_dim, a->page_size, a->page_table_width, kDecodeLongTile);
    if (need_long <= have || noalloc) {
      tile_keys = kDecodeLongTile;
      need = need_long;
    }
  }
  if (noalloc && need > CA_DECODE_NOALLOC_SCRATCH_BYTES) return CA_SCRATCH_EXCEEDED;
  if (!a->q || !a->k_cache || !a->v_cache || !a->lens || !a->page_table || !a->out)
    return CA_DECLINED;
  if ((a->k_new == nullptr) != (a->v_new == nullptr)) return CA_DECLINED;
  if (a->slots && !a->k_new) return CA_DECLINED;
  if (a->new_tokens < 0 || a->new_tokens > (1 << 30) || (a->slots && a->new_tokens > 1)) return CA_DECLINED;
  const int64_t per_seq = a->new_tokens > 1 ? a->new_tokens : 1;
  if (!aligned16(a->q) || !aligned16(a->k_cache) || !aligned16(a->v_cache) ||
      !aligned16(a->out) || !stride16(a->q_stride, a->dtype))
    return CA_DECLINED;
  if (a->k_new && (!aligned16(a->k_new) || !aligned16(a->v_new) || !stride16(a->kv_stride, a->dtype)))
    return CA_DECLINED;
  void* workspace = a->workspace;
  int64_t workspace_bytes = a->workspace_bytes;
  int scratch_device = -1;  // noalloc: the device whose scratch this call uses
  if (noalloc) {
    workspace = nullptr;
    workspace_bytes = 0;
    if (need > 0) {
      const int r = decode_noalloc_scratch(&workspace, &scratch_device);
      if (r != CA_OK) return r;
      workspace_bytes = CA_DECODE_NOALLOC_SCRATCH_BYTES;
    }
  }
  if (need > 0 && (!workspace || !aligned16(workspace) || workspace_bytes < need)) return CA_DECLINED;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t words = a->head_dim * esize(a->dtype) / 4;
  // The reference stores the new token, then attends (paged_attn.mojo:852-863).
  // For a small batch, one token appended at lens (the serving step) is folded
  // into the decode kernel: the wave whose tile holds position lens[s] writes it
  // to the cache and attends it, so one launch does both.  Larger batches,
  // several tokens, or a store at given slots (which need not be the position
  // the row attends) go through a store kernel first: the scatter kernel for one
  // token per sequence (each on a page of its own), the staging one for a prompt.
  const bool fused = a->k_new && !a->slots && per_seq == 1 &&
                     a->num_seqs * a->num_heads <= kFusedAppendMaxRows;
  auto launch = [&]() -> int {
    if (a->k_new && !fused) {
      StoreParams sp{};
      sp.key = static_cast<const uint32_t*>(a->k_new);
      sp.value = static_cast<const uint32_t*>(a->v_new);
      sp.tok_stride_w = a->kv_stride * esize(a->dtype) / 4;
      sp.kc = static_cast<uint32_t*>(a->k_cache);
      sp.vc = static_cast<uint32_t*>(a->v_cache);
      sp.slots = a->slots;
      sp.lens = a->lens;
      sp.page_table = a->page_table;
      sp.pt_width = a->page_table_width;
      sp.ntok = a->num_seqs * per_seq;
      sp.per_seq = per_seq;
      sp.heads = a->num_heads;
      sp.page = a->page_size;
      sp.nblocks = a->num_blocks;
      const int r = per_seq == 1 ? store_scatter_launch(sp, (int)words, st) : store_launch(sp, (int)words, st);
      if (r != CA_OK) return r;
    }

    DecodeParams p{};
    p.q = a->q;
    p.q_stride = a->q_stride;
    p.kc = static_cast<const uint32_t*>(a->k_cache);
    p.vc = a->v_cache;
    p.lens = a->lens;
    // Appending at lens: the row attends lens + 1 keys.  With slots, lens is
    // already the post-store length (_C.mojo:100-103, paged_attn.mojo:721-723).
    p.len_add = (a->k_new && !a->slots) ? (int32_t)per_seq : 0;
    p.page_table = a->page_table;
    p.pt_width = a->page_table_width;
    p.heads = a->num_heads;
    p.page = a->page_size;
    p.nblocks = a->num_blocks;
    p.nseqs = a->num_seqs;
    p.c = a->scale * kLog2e;
    p.tile_keys = tile_keys;
    p.tiles = (int)decode_tiles(a->page_table_width, a->page_size, tile_keys);
    p.slots = decode_workspace_slots(rows, p.tiles);
    const int64_t acc_bytes = decode_acc_bytes(p.slots, a->head_dim);
    p.part_acc = static_cast<float*>(workspace);
    p.part_ml = reinterpret_cast<float*>(static_cast<char*>(workspace) + acc_bytes);
    if (decode_merges(rows, p.slots)) {
      p.counters = reinterpret_cast<uint64_t*>(static_cast<char*>(workspace) + acc_bytes + p.slots * 8);
      p.tag = next_merge_tag();
    }
    p.out = a->out;
    if (fused) {
      p.k_new = static_cast<const uint32_t*>(a->k_new);
      p.v_new = static_cast<const uint32_t*>(a->v_new);
      p.kv_stride_w = a->kv_stride * esize(a->dtype) / 4;
      p.kc_store = static_cast<uint32_t*>(a->k_cache);
      p.vc_store = static_cast<uint32_t*>(a->v_cache);
    }
    return decode_launch(p, (int)a->head_dim, a->dtype == CA_BF16, st);
  };
  // The no-allocation entry's calls that use its one scratch buffer run one after
  // another on the device, whichever streams they come on.
  if (scratch_device >= 0) return decode_noalloc_ordered(scratch_device, st, launch);
  return launch();
}


extern "C" int ca_decode(const ca_decode_args* a, void* stream) { return decode_entry(a, stream, false); }

extern "C" int ca_decode_noalloc(const ca_decode_args* a, void* stream) {
  static_assert(CA_DECODE_NOALLOC_SCRATCH_BYTES == (32ll << 20), "the status string names the size");
  return decode_entry(a, stream, true);
}

extern "C" int64_t ca_flash_workspace_bytes(int64_t batch, int64_t seq_q, int64_t seq_k, int64_t num_heads,
                                            int64_t head_dim, int32_t dtype) {
  if (!dtype_ok(dtype) || !head_dim_ok(head_dim) || batch < 0 || num_heads < 0 || seq_q < 1 || seq_k < 1)
    return 0;
  return flash_rows_workspace_bytes(batch, seq_q, seq_k, num_heads, (int)head_dim, dtype == CA_BF16);
}

extern "C" int ca_flash(const ca_flash_args* a, void* stream) {
  if (!a || !dtype_ok(a->dtype) || !head_dim_ok(a->head_dim)) return CA_DECLINED;
  if (a->batch < 0 || a->num_heads <= 0 || a->seq_q < 1 || a->seq_k < 1) return CA_DECLINED;
  if (a->batch == 0) return CA_OK;
  if (!a->q || !a->k || !a->v || !a->out) return CA_DECLINED;
  if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->out))
    return CA_DECLINED;
  for (int i = 0; i < 3; ++i)
    if (!stride16(a->q_strides[i], a->dtype) || !stride16(a->k_strides[i], a->dtype) ||
        !stride16(a->v_strides[i], a->dtype))
      return CA_DECLINED;
  FlashParams p{};
  p.q = a->q;
  p.k = a->k;
  p.v = a->v;
  p.out = a->out;
  p.batch = a->batch;
  p.seq_q = a->seq_q;
  p.seq_k = a->seq_k;
  p.heads = a->num_heads;
  for (int i = 0; i < 3; ++i) {
    p.qs[i] = a->q_strides[i];
    p.ks[i] = a->k_strides[i];
    p.vs[i] = a->v_strides[i];
  }
  p.c = a->scale * kLog2e;
  p.causal = a->causal ? 1 : 0;
  if (a->workspace_bytes < 0) return CA_DECLINED;
  // The split kernels write their partials with 16-byte stores.
  if (a->workspace && !aligned16(a->workspace) && flash_call_splits(p, (int)a->head_dim, a->dtype == CA_BF16) > 1)
    return CA_DECLINED;
  flash_rows_workspace(p, a->workspace, a->workspace_bytes, (int)a->head_dim, a->dtype == CA_BF16);
  return flash_launch(p, (int)a->head_dim, a->dtype == CA_BF16, static_cast<hipStream_t>(stream));
}

// ---------------------------------------------------------------------------
// Window and sinks, the 8-bit cache, copies of pages
// ---------------------------------------------------------------------------
static bool scale_ok(float scale) { return scale > 0.f && scale < INFINITY; }

// The window in the kernels' terms: no side left open (open: 2^30), and `plain` when it
// leaves nothing out of the causal (or of the full) call.
struct WindowSides {
  int64_t left, right, sinks;
  bool plain, causal;
};
static WindowSides window_sides(int64_t seq_q, int64_t seq_k, bool causal, int64_t left, int64_t right, int64_t sinks) {
  constexpr int64_t kOpen = 1 << 30;
  WindowSides w;
  // The last row stands at seq_k - 1 and sees key 0 with left >= seq_k - 1; the first
  // at seq_k - seq_q and sees the last key with right >= seq_q - 1.
  if (causal) right = 0;
  w.left = left < 0 || left >= seq_k - 1 ? kOpen : left;
  w.right = right < 0 || right >= seq_q - 1 ? kOpen : right;
  w.sinks = sinks < 0 ? 0 : (sinks < seq_k ? sinks : seq_k);
  w.causal = w.right != kOpen;
  w.plain = w.left == kOpen && (w.right == kOpen || w.right == 0);
  return w;
}

static WindowParams window_params(const FlashParams& f, const WindowSides& w) {
  WindowParams p{};
  static_cast<FlashParams&>(p) = f;
  p.left = (int32_t)w.left;
  p.right = (int32_t)w.right;
  p.sinks = (int32_t)w.sinks;
  return p;
}

// What a window call's workspace holds: the partials of `slots` (row, split) pairs, then the
// `words` of an fp32 call on split operands.
struct WindowSpace {
  int64_t splits, slots, words, bytes;
};
static WindowSpace window_space(const WindowParams& p, int64_t head_dim, int32_t dtype) {
  const WinF32Blocks f = dtype == CA_BF16 ? WinF32Blocks{0, 1, false} : flash_window_f32_blocks(p, (int)head_dim);
  WindowSpace w{f.splits, 0, f.blocks * f.splits, 0};
  if (f.blocks == 0) w.splits = dtype == CA_BF16 ? flash_window_bf16_splits(p) : flash_window_f32_splits(p, (int)head_dim);
  if (w.splits > 1) w.slots = p.batch * p.heads * p.seq_q * w.splits;
  w.bytes = w.slots * (head_dim + 2) * 4 + w.words * 4;
  return w;
}

extern "C" int64_t ca_flash_window_workspace_bytes(int64_t batch, int64_t seq_q, int64_t seq_k, int64_t num_heads,
                                                   int64_t head_dim, int32_t dtype, int32_t causal, int64_t left,
                                                   int64_t right, int64_t sinks) {
  if (!dtype_ok(dtype) || !head_dim_ok(head_dim) || batch < 1 || num_heads < 1 || seq_q < 1 || seq_k < 1) return 0;
  if (seq_q > kWindowMaxSeq || seq_k > kWindowMaxSeq) return 0;  // declined
  const WindowSides w = window_sides(seq_q, seq_k, causal != 0, left, right, sinks);
  if (w.plain) return ca_flash_workspace_bytes(batch, seq_q, seq_k, num_heads, head_dim, dtype);
  FlashParams f{};
  f.batch = batch;
  f.seq_q = seq_q;
  f.seq_k = seq_k;
  f.heads = num_heads;
  return window_space(window_params(f, w), head_dim, dtype).bytes;
}

extern "C" int ca_flash_window(const ca_flash_window_args* wa, void* stream) {
  if (!wa) return CA_DECLINED;
  const ca_flash_args* a = &wa->flash;
  if (!dtype_ok(a->dtype) || !head_dim_ok(a->head_dim) || wa->sinks < 0 || !scale_ok(a->scale)) return CA_DECLINED;
  if (a->batch < 0 || a->num_heads <= 0 || a->seq_q < 1 || a->seq_k < 1) return CA_DECLINED;
  if (a->seq_q > kWindowMaxSeq || a->seq_k > kWindowMaxSeq) return CA_DECLINED;
  const WindowSides w = window_sides(a->seq_q, a->seq_k, a->causal != 0, wa->left, wa->right, wa->sinks);
  if (w.plain) {
    ca_flash_args f = *a;
    f.causal = w.causal ? 1 : 0;
    return ca_flash(&f, stream);
  }
  if (a->batch == 0) return CA_OK;
  if (!a->q || !a->k || !a->v || !a->out) return CA_DECLINED;
  if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->out)) return CA_DECLINED;
  for (int i = 0; i < 3; ++i)
    if (!stride16(a->q_strides[i], a->dtype) || !stride16(a->k_strides[i], a->dtype) || !stride16(a->v_strides[i], a->dtype))
      return CA_DECLINED;
  FlashParams f{};
  f.q = a->q;
  f.k = a->k;
  f.v = a->v;
  f.out = a->out;
  f.batch = a->batch;
  f.seq_q = a->seq_q;
  f.seq_k = a->seq_k;
  f.heads = a->num_heads;
  for (int i = 0; i < 3; ++i) {
    f.qs[i] = a->q_strides[i];
    f.ks[i] = a->k_strides[i];
    f.vs[i] = a->v_strides[i];
  }
  f.c = a->scale * kLog2e;
  WindowParams p = window_params(f, w);
  const WindowSpace ws = window_space(p, a->head_dim, a->dtype);
  if (ws.bytes > 0) {
    if (!a->workspace || !aligned16(a->workspace) || a->workspace_bytes < ws.bytes) return CA_DECLINED;
    p.part_acc = static_cast<float*>(a->workspace);
    p.part_ml = p.part_acc + ws.slots * a->head_dim;
    p.workspace_bytes = a->workspace_bytes;
    if (ws.words > 0) {
      p.redo = reinterpret_cast<int32_t*>(p.part_ml + 2 * ws.slots);
      p.redo_splits = (int32_t)ws.splits;
    }
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (a->dtype == CA_BF16) return flash_window_bf16_launch(p, (int)a->head_dim, st);
  if (ws.words > 0) {
    const int r = flash_window_split_launch(p, (int)a->head_dim, st);
    if (r != CA_OK) return r;
  }
  return flash_window_f32_launch(p, (int)a->head_dim, st);
}

static int64_t win_left(int64_t left, int64_t cap) { return left < 0 || left >= cap ? -1 : left; }

// Window and 8-bit decodes whose split rows are merged by their last block inside the
// kernel: up to 512 rows of 4 blocks, or 32 rows of 8.  Second launch / in-kernel, us per
// call with a one-token append, bf16 unless noted: 8 rows E=64, 2 blocks 10.3 / 7.9, 8 blocks 9.3 /
// 8.4, 16 blocks 10.9 / 11.5, 63 blocks 21.8 / 36; 32 rows E=128, 3 blocks 12.2 / 10.6, 4
// blocks 12.7 / 11.4 (8-bit 11.1 / 9.8), 8 blocks 16.6 / 16.0, E=64 16 blocks 16.9 / 23; 64 rows
// 7 blocks E=64 15.8 / 16.8, E=128 24.3 / 23.6; 128 rows E=64 5 blocks 19.4 / 19.8; 512 rows
// 4 blocks 78.2 / 78.2, 5 blocks E=64 55.2 / 56.9; 1024 rows E=64, 3 blocks 63.3 / 64.2.
static bool win_decode_merges(int64_t rows, int64_t slots) {
  return slots > 0 && rows <= kMergeMaxRows && slots <= rows * (rows <= 32 ? 8 : kMergeMaxBlocks);
}

static int64_t win_decode_ws_bytes(int64_t rows, int64_t slots, int64_t head_dim) {
  return decode_acc_bytes(slots, head_dim) + slots * 8 + (win_decode_merges(rows, slots) ? rows * 8 : 0);
}

extern "C" int64_t ca_decode_window_workspace_bytes(int64_t num_seqs, int64_t num_heads, int64_t head_dim,
                                                    int64_t page_size, int64_t page_table_width, int64_t left,
                                                    int64_t sinks) {
  if (num_seqs < 0 || num_heads < 0 || page_size <= 0 || page_table_width < 0 || sinks < 0) return -1;
  const int64_t cap = page_table_width * page_size;
  const int64_t tiles = win_decode_tiles(page_table_width, page_size, win_left(left, cap), sinks < cap ? sinks : cap);
  // One tile more: an 8-bit cache's last page, if the call appends to it.
  const int64_t rows = num_seqs * num_heads;
  return win_decode_ws_bytes(rows, win_decode_slots(rows, tiles + 1), head_dim);
}

extern "C" int ca_decode_window(const ca_decode_window_args* wa, void* stream) {
  if (!wa) return CA_DECLINED;
  const ca_decode_args* a = &wa->decode;
  if (!dtype_ok(a->dtype) || !head_dim_ok(a->head_dim) || !page_ok(a->page_size) || wa->sinks < 0 || !scale_ok(a->scale))
    return CA_DECLINED;
  if (a->num_seqs < 0 || a->num_heads <= 0 || a->num_blocks < 0 || a->page_table_width < 0) return CA_DECLINED;
  if ((wa->k_scale == nullptr) != (wa->v_scale == nullptr) || a->slots) return CA_DECLINED;
  if ((uintptr_t)wa->longest % 8) return CA_DECLINED;
  if ((a->k_new == nullptr) != (a->v_new == nullptr) || a->new_tokens < 0 || a->new_tokens > (1 << 30)) return CA_DECLINED;
  if (a->num_seqs == 0) return CA_OK;
  // An empty page table or cache is never read: its pointer may be null.
  if (!a->q || !a->lens || !a->out || (a->page_table_width > 0 && !a->page_table) ||
      (a->num_blocks > 0 && (!a->k_cache || !a->v_cache)))
    return CA_DECLINED;
  if (!aligned16(a->q) || !aligned16(a->k_cache) || !aligned16(a->v_cache) || !aligned16(a->out) ||
      !stride16(a->q_stride, a->dtype))
    return CA_DECLINED;
  if (a->k_new && (!aligned16(a->k_new) || !aligned16(a->v_new) || !stride16(a->kv_stride, a->dtype))) return CA_DECLINED;
  const bool f8 = wa->k_scale != nullptr;
  const int64_t rows = a->num_seqs * a->num_heads, cap = a->page_table_width * a->page_size;
  const int64_t per_seq = a->new_tokens > 1 ? a->new_tokens : 1;
  WinDecodeParams p{};
  p.left = win_left(wa->left, cap);
  p.sinks = wa->sinks < cap ? wa->sinks : cap;
  p.longest = wa->longest;
  const bool fold = a->k_new && per_seq == 1 && win_decode_folds(rows, a->page_size, f8);
  const int64_t tiles = win_decode_tiles(a->page_table_width, a->page_size, p.left, p.sinks) + (fold && f8 ? 1 : 0);
  if (tiles > 0x7fffffff) return CA_DECLINED;
  p.tiles = (int)tiles;
  p.slots = win_decode_slots(rows, p.tiles);
  if (p.slots > 0 && (!a->workspace || !aligned16(a->workspace) ||
                      a->workspace_bytes < win_decode_ws_bytes(rows, p.slots, a->head_dim)))
    return CA_DECLINED;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (p.longest) {  // a replayed graph would tell a host that no longer listens
    if (a->k_new && !fold) return CA_DECLINED;
    hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(st, &capture) != hipSuccess || capture != hipStreamCaptureStatusNone) return CA_DECLINED;
  }
  // One new token per sequence is stored by the decode itself in small calls, others go in
  // first, by a kernel of their own.
  if (fold) {
    p.k_new = static_cast<const uint32_t*>(a->k_new);
    p.v_new = static_cast<const uint32_t*>(a->v_new);
    p.new_stride = a->kv_stride;
    p.kc_store = static_cast<uint32_t*>(a->k_cache);
    p.vc_store = static_cast<uint32_t*>(a->v_cache);
    p.k_scale_store = wa->k_scale;
    p.v_scale_store = wa->v_scale;
  } else if (a->k_new) {
    int r;
    if (f8) {
      Store8Params sp{};
      sp.key = a->k_new;
      sp.value = a->v_new;
      sp.tok_stride = a->kv_stride;
      sp.kc = static_cast<uint32_t*>(a->k_cache);
      sp.vc = static_cast<uint32_t*>(a->v_cache);
      sp.k_scale = wa->k_scale;
      sp.v_scale = wa->v_scale;
      sp.lens = a->lens;
      sp.page_table = a->page_table;
      sp.pt_width = a->page_table_width;
      sp.ntok = a->num_seqs * per_seq;
      sp.per_seq = per_seq;
      sp.heads = a->num_heads;
      sp.page = a->page_size;
      sp.nblocks = a->num_blocks;
      r = store8_launch(sp, (int)a->head_dim, a->dtype == CA_BF16, st);
    } else {
      const int64_t words = a->head_dim * esize(a->dtype) / 4;
      StoreParams sp{};
      sp.key = static_cast<const uint32_t*>(a->k_new);
      sp.value = static_cast<const uint32_t*>(a->v_new);
      sp.tok_stride_w = a->kv_stride * esize(a->dtype) / 4;
      sp.kc = static_cast<uint32_t*>(a->k_cache);
      sp.vc = static_cast<uint32_t*>(a->v_cache);
      sp.lens = a->lens;
      sp.page_table = a->page_table;
      sp.pt_width = a->page_table_width;
      sp.ntok = a->num_seqs * per_seq;
      sp.per_seq = per_seq;
      sp.heads = a->num_heads;
      sp.page = a->page_size;
      sp.nblocks = a->num_blocks;
      r = per_seq == 1 ? store_scatter_launch(sp, (int)words, st) : store_launch(sp, (int)words, st);
    }
    if (r != CA_OK) return r;
  }
  p.q = a->q;
  p.q_stride = a->q_stride;
  p.kc = static_cast<const uint32_t*>(a->k_cache);
  p.vc = a->v_cache;
  p.lens = a->lens;
  p.len_add = a->k_new ? (int32_t)per_seq : 0;
  p.page_table = a->page_table;
  p.pt_width = a->page_table_width;
  p.heads = a->num_heads;
  p.page = a->page_size;
  p.nblocks = a->num_blocks;
  p.nseqs = a->num_seqs;
  p.c = a->scale * kLog2e;
  p.part_acc = static_cast<float*>(a->workspace);
  p.part_ml = reinterpret_cast<float*>(static_cast<char*>(a->workspace) + decode_acc_bytes(p.slots, a->head_dim));
  if (win_decode_merges(rows, p.slots)) {
    p.counters = reinterpret_cast<uint64_t*>(p.part_ml + 2 * p.slots);
    p.tag = next_merge_tag();
  }
  p.out = a->out;
  p.k_scale = wa->k_scale;
  p.v_scale = wa->v_scale;
  return win_decode_launch(p, (int)a->head_dim, a->dtype == CA_BF16, st);
}

extern "C" int64_t ca_store_fp8_workspace_bytes(int64_t num_tokens, int64_t num_blocks, int64_t page_size) {
  if (num_tokens < 0 || num_blocks < 0 || page_size <= 0) return -1;
  return store8_work_ints(num_tokens, num_blocks, page_size) * 4;
}

extern "C" int ca_store_fp8(const ca_store_fp8_args* sa, void* stream) {
  if (!sa) return CA_DECLINED;
  const ca_store_args* a = &sa->store;
  if (!dtype_ok(a->dtype) || !head_dim_ok(a->head_dim) || !page_ok(a->page_size)) return CA_DECLINED;
  if (a->num_tokens < 0 || a->num_heads <= 0 || a->num_blocks < 0) return CA_DECLINED;
  if (a->num_tokens == 0) return CA_OK;
  if (!a->key || !a->value || !a->k_cache || !a->v_cache || !a->slot_mapping || !sa->k_scale || !sa->v_scale)
    return CA_DECLINED;
  if (!aligned16(a->key) || !aligned16(a->value) || !aligned16(a->k_cache) || !aligned16(a->v_cache)) return CA_DECLINED;
  const bool one = a->num_tokens == 1;  // its stride is not read
  if (!one && (!stride16(a->token_stride, a->dtype) || a->token_stride < a->num_heads * a->head_dim)) return CA_DECLINED;
  const int64_t need = ca_store_fp8_workspace_bytes(a->num_tokens, a->num_blocks, a->page_size);
  if (need > 0 && (!sa->workspace || !aligned16(sa->workspace) || sa->workspace_bytes < need)) return CA_DECLINED;
  Store8Params p{};
  p.key = a->key;
  p.value = a->value;
  p.tok_stride = one ? 0 : a->token_stride;
  p.kc = static_cast<uint32_t*>(a->k_cache);
  p.vc = static_cast<uint32_t*>(a->v_cache);
  p.k_scale = sa->k_scale;
  p.v_scale = sa->v_scale;
  p.slots = a->slot_mapping;
  p.ntok = a->num_tokens;
  p.per_seq = 1;
  p.heads = a->num_heads;
  p.page = a->page_size;
  p.nblocks = a->num_blocks;
  p.work = static_cast<int32_t*>(sa->workspace);
  return store8_launch(p, (int)a->head_dim, a->dtype == CA_BF16, static_cast<hipStream_t>(stream));
}

extern "C" int ca_copy_blocks(const ca_copy_blocks_args* a, void* stream) {
  if (!a || a->num_caches < 0 || a->num_scales < 0 || a->num_pairs < 0 || a->num_blocks < 0) return CA_DECLINED;
  if (a->num_caches > 0 && (a->block_bytes <= 0 || a->block_bytes % 16)) return CA_DECLINED;
  if (a->num_scales > 0 && (a->row_bytes <= 0 || a->row_bytes % 4)) return CA_DECLINED;
  const int64_t arrays = a->num_caches + a->num_scales;
  if (arrays == 0 || a->num_pairs == 0) return CA_OK;
  if ((a->num_caches > 0 && !a->caches) || (a->num_scales > 0 && !a->scales) || !a->mapping) return CA_DECLINED;
  auto array = [&](int64_t i) { return i < a->num_caches ? a->caches[i] : a->scales[i - a->num_caches]; };
  for (int64_t i = 0; i < arrays; ++i)
    if (!array(i) || ((uintptr_t)array(i) & (i < a->num_caches ? 15 : 3))) return CA_DECLINED;
  CopyParams p{};
  p.mapping = a->mapping;
  p.pairs = a->num_pairs;
  p.nblocks = a->num_blocks;
  p.bytes = a->num_caches > 0 ? a->block_bytes : 16;  // scales alone: one piece each
  p.row_bytes = a->row_bytes;
  for (int64_t i = 0; i < arrays; i += kCopyArrays) {
    p.arrays = (int)(arrays - i < kCopyArrays ? arrays - i : kCopyArrays);
    p.caches = (int)(a->num_caches - i < 0 ? 0 : (a->num_caches - i < p.arrays ? a->num_caches - i : p.arrays));
    for (int k = 0; k < p.arrays; ++k) p.base[k] = array(i + k);
    const int r = copy_launch(p, static_cast<hipStream_t>(stream));
    if (r != CA_OK) return r;
  }
  return CA_OK;
}
