// Host side of the C ABI: parameter checks, operand address resolution, host /
// device pointer classification with staging, kernel selection and launch.
//
// The checks restate the reference's debug-build assertions
// (mmt4d.c:12-48, pack.c:51-103, unpack.c:31-81) and are always on here: a
// rejected call costs microseconds next to a kernel launch, and an out-of-range
// parameter reaching a GPU kernel can fault the device rather than one process.
#include <algorithm>
#include <atomic>
#include <chrono>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <immintrin.h>

#include "host_crew.h"
#include "uk_internal.h"

#define UK_API extern "C" __attribute__((visibility("default")))

// Default failure handler; an embedder's strong definition replaces it.
extern "C" __attribute__((visibility("default"), weak)) void iree_uk_assert_fail(
    const char* file, int line, const char* function, const char* condition) {
  fflush(stdout);
  fprintf(stderr, "%s:%d: %s: iree_uk_mi355x check failed: %s\n", file, line, function, condition);
  fflush(stderr);
  abort();
}

namespace uk {
hipError_t launch_pack_generic(const PackArgs& a, hipStream_t stream, const char** name);
hipError_t launch_unpack_generic(const UnpackArgs& a, hipStream_t stream, const char** name);
}  // namespace uk

namespace {

thread_local hipStream_t tl_stream = nullptr;
thread_local bool tl_async = false;
thread_local const char* tl_last_kernel = "";
std::atomic<iree_uk_mi355x_fail_handler_t> g_fail_handler{nullptr};

void report_failure(const char* file, int line, const char* function, const char* condition) {
  iree_uk_mi355x_fail_handler_t h = g_fail_handler.load(std::memory_order_acquire);
  if (h) {
    h(file, line, function, condition);
  } else {
    iree_uk_assert_fail(file, line, function, condition);
  }
}

// Checks a parameter condition; on failure reports it and leaves the entry
// point (which returns void) without launching anything.
#define UK_REQUIRE(cond)                                      \
  do {                                                        \
    if (!(cond)) {                                            \
      report_failure(__FILE__, __LINE__, __func__, #cond);    \
      return;                                                 \
    }                                                         \
  } while (0)

// The same in a function that returns whether its checks hold.
#define UK_REQUIRE_TRUE(cond)                                 \
  do {                                                        \
    if (!(cond)) {                                            \
      report_failure(__FILE__, __LINE__, __func__, #cond);    \
      return false;                                           \
    }                                                         \
  } while (0)

// Checks a HIP call inside a function returning bool (true = ok).
#define UK_HIP_OK(expr)                                                       \
  do {                                                                        \
    hipError_t uk_err_ = (expr);                                              \
    if (uk_err_ != hipSuccess) {                                              \
      char uk_msg_[256];                                                      \
      snprintf(uk_msg_, sizeof uk_msg_, "%s -> %s", #expr, hipGetErrorString(uk_err_)); \
      report_failure(__FILE__, __LINE__, __func__, uk_msg_);                  \
      return false;                                                           \
    }                                                                         \
  } while (0)

// outer * tile >= size for non-negative values, without forming a product
// that may not fit.
bool tiles_cover(int64_t outer, int64_t tile, int64_t size) {
  if (size == 0) return true;
  if (outer == 0 || tile == 0) return false;
  return outer >= size / tile + (size % tile != 0);
}

bool in_unsigned_range(int64_t v, int bits) { return v >= 0 && v < ((int64_t)1 << bits); }

// True if a kernel on the current device may dereference `p`.
bool device_accessible(const void* p) {
  hipPointerAttribute_t attr;
  hipError_t e = hipPointerGetAttributes(&attr, p);
  if (e != hipSuccess) {
    (void)hipGetLastError();  // plain host memory is reported as an error
    return false;
  }
  return attr.type == hipMemoryTypeDevice || attr.type == hipMemoryTypeManaged ||
         attr.type == hipMemoryTypeHost;
}

// Per-thread device memory that host operands are mirrored in (grow-only, released when the thread exits or goes on to
// another device).
struct StageArena {
  uint8_t* ptr = nullptr;
  size_t capacity = 0;
  int device = -1;
  ~StageArena() {
    // At process teardown the HIP runtime may already be gone: errors are moot.
    if (ptr) (void)hipFree(ptr);
  }
};
thread_local StageArena tl_arena;

// Per-thread pinned memory that host operands pass through on their way to and from the device: the CPU copies the
// caller's pages (55 to 80 GB/s) a chunk at a time while the previous chunks are on the bus (50 GB/s each way). The
// runtime's own path for pageable memory moves 20 to 33 GB/s up and 17 down, in 30 to 100 us for a few KiB. int8 through
// both: 64 x 256 x 256 47 -> 21 us, 512 x 2048 x 2048 (5 MB up, 4 down) 430 -> 255, 4096 x 2048 x 4096 2731 -> 1458.
//
// It is as large as the largest call of the thread so far needs, 64 KiB to 8 MiB. Operands that together fit go up from
// their place in it; larger ones through its eight slots in turn, each of them guarded by an event.
struct HostPipe {
  static constexpr size_t kSlotBytes = 1 << 20, kFirstBytes = 128 << 10;
  static constexpr int kSlots = 8;
  static constexpr size_t kMostBytes = kSlots * kSlotBytes, kLeastBytes = 64 << 10;
  static constexpr size_t kHalfBytes = kMostBytes / 2;  // a download of more than this alternates between halves
  static constexpr int kFlags = (int)(kMostBytes / uk::kDownloadPieceBytes);
  static constexpr size_t kFlagBytes = 4096;
  static_assert(kFlags * sizeof(uint32_t) <= kFlagBytes, "room for the flags");
  uint32_t* flags = nullptr;  // at the start of the allocation
  uint8_t* pinned = nullptr;  // behind them
  size_t capacity = 0;
  uint32_t generation = 0;
  hipEvent_t event[kSlots] = {};  // exist where a call has needed them
  int device = -1;

  ~HostPipe() { release(); }
  void release() {
    for (hipEvent_t& e : event) {
      if (e) (void)hipEventDestroy(e);
      e = nullptr;
    }
    if (flags) (void)hipHostFree(flags);
    flags = nullptr;
    pinned = nullptr;
    capacity = 0;
  }
  // For a call that mirrors `bytes` in all. False: no pinned memory to be had; the caller copies from pageable memory.
  bool ready(int current_device, size_t bytes) {
    const bool slots = bytes > kMostBytes;
    if (!pinned || device != current_device || capacity < (slots ? kMostBytes : bytes)) {
      release();
      device = current_device;
      size_t size = kLeastBytes;
      while (size < kMostBytes && size < bytes) size *= 2;
      void* block = nullptr;
      if (hipHostMalloc(&block, kFlagBytes + size, hipHostMallocDefault) != hipSuccess) {
        (void)hipGetLastError();
        return false;
      }
      flags = (uint32_t*)block;
      pinned = (uint8_t*)block + kFlagBytes;
      capacity = size;
      memset(flags, 0, kFlagBytes);
      generation = 0;
    }
    for (hipEvent_t& e : event) {
      if (!slots || e) continue;
      if (hipEventCreateWithFlags(&e, hipEventDisableTiming) != hipSuccess) {
        (void)hipGetLastError();
        e = nullptr;
        release();
        return false;
      }
    }
    return true;
  }
};
thread_local HostPipe tl_pipe;

// Static staging memory of the allocation-free entry point: one array per
// device, owned by the code object, resolved to a device address once per
// device (the array's name is only a host-side handle for that lookup).
constexpr size_t kScratchBytes = (size_t)IREE_UK_MI355X_NOALLOC_MAX_STAGED_BYTES;
constexpr int kMaxDevices = 64;
static __device__ __align__(256) unsigned char scratch[kScratchBytes];
std::atomic<unsigned char*> g_scratch_ptr[kMaxDevices];
// One call at a time may stage host operands in a device's array: taken with a
// try-lock (a second caller is told so instead of waiting or corrupting the
// first one's operands), held until the call's results are back on the host.
std::atomic<bool> g_scratch_busy[kMaxDevices];

struct ScratchLease {
  std::atomic<bool>* flag = nullptr;
  ScratchLease() = default;
  ScratchLease(const ScratchLease&) = delete;
  ScratchLease& operator=(const ScratchLease&) = delete;
  ~ScratchLease() {
    if (flag) flag->store(false, std::memory_order_release);
  }
};

// Device address of the current device's `scratch` (nullptr after reporting
// a failure).
unsigned char* scratch_for_current_device(int* device_out = nullptr) {
  int device = -1;
  if (hipGetDevice(&device) != hipSuccess || device < 0 || device >= kMaxDevices) {
    (void)hipGetLastError();
    return nullptr;
  }
  if (device_out) *device_out = device;
  unsigned char* ptr = g_scratch_ptr[device].load(std::memory_order_acquire);
  if (ptr) return ptr;
  void* resolved = nullptr;
  if (hipGetSymbolAddress(&resolved, HIP_SYMBOL(scratch)) != hipSuccess || !resolved) {
    (void)hipGetLastError();
    return nullptr;
  }
  // Two threads racing here resolve the same address.
  g_scratch_ptr[device].store((unsigned char*)resolved, std::memory_order_release);
  return (unsigned char*)resolved;
}

// Where the calling entry point mirrors host operands: the thread's grow-only memory (may call hipMalloc), or the
// device's static scratch (never allocates; fails when the operands do not fit).
struct Stager {
  bool no_alloc = false;
  bool copies_issued = false;           // something was enqueued on the stream for this call
  bool piped = false;                   // contiguous operands go through the thread's pinned memory
  uk::HostCrew* crew = nullptr;         // helps with those copies, until the end of the call
  ScratchLease lease;                   // held while the static scratch is in use
  ~Stager() {
    if (crew) crew->release();
  }
};

size_t rounded_for_staging(size_t bytes) { return (bytes + 255) & ~(size_t)255; }

bool stage_reserve(Stager& stager, size_t bytes, uint8_t** out) {
  int device = -1;
  if (stager.no_alloc) {
    if (bytes > kScratchBytes) {
      report_failure(__FILE__, __LINE__, __func__,
                     "host operands exceed IREE_UK_MI355X_NOALLOC_MAX_STAGED_BYTES of static staging memory");
      return false;
    }
    unsigned char* base = scratch_for_current_device(&device);
    if (!base) {
      report_failure(__FILE__, __LINE__, __func__, "hipGetSymbolAddress(scratch) failed on the current device");
      return false;
    }
    bool expected = false;
    if (!g_scratch_busy[device].compare_exchange_strong(expected, true, std::memory_order_acq_rel)) {
      report_failure(__FILE__, __LINE__, __func__,
                     "static staging memory busy: another iree_uk_mi355x_mmt4d_noalloc_p call with host "
                     "operands is running on this device");
      return false;
    }
    stager.lease.flag = &g_scratch_busy[device];
    *out = base;
    return true;
  }
  UK_HIP_OK(hipGetDevice(&device));
  StageArena& s = tl_arena;
  if (s.capacity < bytes || s.device != device) {
    if (s.ptr) UK_HIP_OK(hipFree(s.ptr));
    s.ptr = nullptr;
    s.capacity = 0;
    size_t cap = bytes + bytes / 4 + 256;
    UK_HIP_OK(hipMalloc((void**)&s.ptr, cap));
    s.capacity = cap;
    s.device = device;
  }
  stager.piped = tl_pipe.ready(device, bytes);
  *out = s.ptr;
  return true;
}

// int64 arithmetic on caller-provided sizes that records overflow instead of
// wrapping (the checks of the reference admit sizes whose products do not fit).
struct Checked {
  bool ok = true;
  int64_t mul(int64_t a, int64_t b) {
    int64_t r = 0;
    if (__builtin_mul_overflow(a, b, &r)) ok = false;
    return ok ? r : 0;
  }
  int64_t add(int64_t a, int64_t b) {
    int64_t r = 0;
    if (__builtin_add_overflow(a, b, &r)) ok = false;
    return ok ? r : 0;
  }
  // Bytes of `elems` elements of `bits` bits each (sub-byte types: the callers
  // have checked that the count is a whole number of bytes).
  int64_t bytes(int64_t elems, int bits) { return bits >= 8 ? mul(elems, bits / 8) : elems / (8 / bits); }
};

// `base + bytes` without the undefined behaviour of pointer arithmetic outside
// an object: callers may pass `allocation - offset` as the base.
const uint8_t* offset_pointer(const void* base, int64_t bytes) {
  return (const uint8_t*)((uintptr_t)base + (uintptr_t)bytes);
}

// A strided set of rows inside one operand: `rows` rows of `width` bytes,
// `pitch` bytes apart; `span` is the byte count from the first to the last
// touched byte.
struct RowRegion {
  int64_t rows = 0, width = 0, pitch = 0, span = 0;
};

RowRegion make_region(Checked& c, int64_t rows, int64_t width, int64_t pitch) {
  RowRegion r;
  r.rows = rows; r.width = width; r.pitch = pitch;
  r.span = rows <= 0 || width <= 0 ? 0 : c.add(c.mul(rows - 1, pitch), width);
  return r;
}

// The same bytes as one row (for operands whose rows overlap or interleave).
RowRegion as_one_span(const RowRegion& r) {
  RowRegion o;
  o.rows = 1; o.width = r.span; o.pitch = 0; o.span = r.span;
  return o;
}

bool copy_rows(void* dst, const void* src, const RowRegion& r, hipMemcpyKind kind, hipStream_t s) {
  if (r.span == 0) return true;
  if (r.rows == 1 || r.pitch == r.width) {
    UK_HIP_OK(hipMemcpyAsync(dst, src, (size_t)r.span, kind, s));
  } else {
    UK_HIP_OK(hipMemcpy2DAsync(dst, (size_t)r.pitch, src, (size_t)r.pitch, (size_t)r.width,
                               (size_t)r.rows, kind, s));
  }
  return true;
}

// One operand of a call. For a host operand the region is mirrored at the same layout in device memory; `upload` says
// whether its current contents are needed there.
struct Operand {
  const void* ptr;
  RowRegion region;
  bool upload;
  const void* dev = nullptr;   // where the kernel finds it
  const void* host = nullptr;  // non-null iff mirrored
  bool contiguous() const { return region.rows == 1 || region.pitch == region.width; }
};

// Copies between the caller's memory and the pinned memory. `stream_past_caches` (operands that together are larger than
// what the caches are likely to hold anyway): 42 GB/s on cold pages where memcpy moves 33, both ways.
__attribute__((target("avx2"))) void copy_past_caches(uint8_t* dst, const uint8_t* src, size_t n) {
  const size_t head = (size_t)(-(uintptr_t)dst & 31);
  if (n < 256) {
    memcpy(dst, src, n);
    return;
  }
  memcpy(dst, src, head);
  dst += head; src += head; n -= head;
  for (; n >= 128; n -= 128, dst += 128, src += 128) {
    _mm_prefetch((const char*)src + 1024, _MM_HINT_NTA);
    _mm_prefetch((const char*)src + 1088, _MM_HINT_NTA);
    const __m256i a = _mm256_loadu_si256((const __m256i*)src), b = _mm256_loadu_si256((const __m256i*)(src + 32)),
                  c = _mm256_loadu_si256((const __m256i*)(src + 64)), d = _mm256_loadu_si256((const __m256i*)(src + 96));
    _mm256_stream_si256((__m256i*)dst, a);
    _mm256_stream_si256((__m256i*)(dst + 32), b);
    _mm256_stream_si256((__m256i*)(dst + 64), c);
    _mm256_stream_si256((__m256i*)(dst + 96), d);
  }
  _mm_sfence();
  memcpy(dst, src, n);
}

constexpr size_t kPastCachesBytes = 2 << 20;
void host_copy(void* dst, const void* src, size_t n, bool stream_past_caches) {
  static const bool avx2 = __builtin_cpu_supports("avx2");
  if (stream_past_caches && avx2) copy_past_caches((uint8_t*)dst, (const uint8_t*)src, n);
  else memcpy(dst, src, n);
}

// Contiguous operands, mirrored one after the other from `base` on, to the device through the pinned memory: chunks
// that double from 128 KiB to 1 MiB (the first one is on the bus early, the later ones cost few launches), small
// operands together in one.
bool pipe_up(Stager& stager, uint8_t* base, Operand* const* ops, int count, hipStream_t stream) {
  HostPipe& pipe = tl_pipe;
  const Operand& last = *ops[count - 1];
  const size_t total = (size_t)((const uint8_t*)last.dev - base) + (size_t)last.region.span;
  const bool slots = total > HostPipe::kMostBytes, past_caches = total >= kPastCachesBytes;
  constexpr size_t kPiece = 64 << 10;  // of a chunk, per helper and turn
  size_t chunk = HostPipe::kFirstBytes;
  for (size_t at = 0, n = 0, used = 0; at < total; at += n, ++used) {
    const int slot = (int)(used % HostPipe::kSlots);
    if (slots && used >= (size_t)HostPipe::kSlots) UK_HIP_OK(hipEventSynchronize(pipe.event[slot]));
    n = total - at < chunk ? total - at : chunk;
    uint8_t* const place = pipe.pinned + (slots ? (size_t)slot * HostPipe::kSlotBytes : at);
    auto fill = [&](size_t from, size_t to) {  // of the mirrored bytes
      for (int op = 0; op < count; ++op) {
        const size_t begin = (size_t)((const uint8_t*)ops[op]->dev - base), end = begin + (size_t)ops[op]->region.span;
        const size_t f = begin > from ? begin : from, t = end < to ? end : to;
        if (f < t) host_copy(place + (f - at), (const uint8_t*)ops[op]->host + (f - begin), t - f, past_caches);
      }
    };
    if (stager.crew && n > kPiece) {
      stager.crew->run((uint32_t)((n + kPiece - 1) / kPiece), [&](uint32_t i) {
        const size_t from = at + i * kPiece;
        fill(from, from + kPiece < at + n ? from + kPiece : at + n);
      }, [] {});
    } else {
      fill(at, at + n);
    }
    UK_HIP_OK(uk::launch_upload(place, base + at, n, stream));
    if (slots) UK_HIP_OK(hipEventRecord(pipe.event[slot], stream));
    if (chunk < HostPipe::kSlotBytes) chunk *= 2;
  }
  return true;
}

// The way back, results visible on return. The pinned memory is used in halves: while the pieces of one are taken as
// their flags come in, the other is filled. (Everything that the caller's stream did before has ended with the last flag.)
bool pipe_down(const Stager& stager, void* host, const void* dev, size_t bytes, hipStream_t stream) {
  HostPipe& pipe = tl_pipe;
  constexpr size_t kHalf = HostPipe::kHalfBytes, kPiece = uk::kDownloadPieceBytes;
  const uint32_t first_generation = pipe.generation + 1;
  pipe.generation += (uint32_t)((bytes + kHalf - 1) / kHalf);
  std::atomic<bool> failed{false};
  hipError_t status = hipSuccess;
  auto send = [&](size_t at) -> bool {
    const size_t half = at / kHalf % 2, n = bytes - at < kHalf ? bytes - at : kHalf;
    UK_HIP_OK(uk::launch_download((const uint8_t*)dev + at, pipe.pinned + half * kHalf, pipe.flags + half * (kHalf / kPiece),
                                  first_generation + (uint32_t)(at / kHalf), n, stream));
    return true;
  };
  const std::thread::id caller = std::this_thread::get_id();
  if (!send(0)) return false;
  for (size_t at = 0; at < bytes && !failed; at += kHalf) {
    if (at + kHalf < bytes && !send(at + kHalf)) return false;  // (into the half that was taken before this one)
    const size_t half = at / kHalf % 2, n = bytes - at < kHalf ? bytes - at : kHalf;
    const uint32_t generation = first_generation + (uint32_t)(at / kHalf);
    const uint32_t* flags = pipe.flags + half * (kHalf / kPiece);
    const uint32_t pieces = (uint32_t)((n + kPiece - 1) / kPiece);
    // A stream that has ended (or failed) without setting its flags will not set them any more.
    auto check_stream = [&] {
      const hipError_t e = hipStreamQuery(stream);
      if (e == hipErrorNotReady) return;
      if (e == hipSuccess && __atomic_load_n(flags + pieces - 1, __ATOMIC_ACQUIRE) == generation) return;
      status = e;
      failed = true;
    };
    if (at == 0) {
      // The first piece comes when everything that the stream had before has ended, the product among it. That is polled
      // for while it may be a matter of microseconds; then the thread sleeps between looks, a sixteenth of what it has
      // waited (half a millisecond at most), and the helpers sleep.
      typedef std::chrono::steady_clock clock;
      const clock::time_point start = clock::now();
      for (uint32_t spins = 1; __atomic_load_n(flags, __ATOMIC_ACQUIRE) != generation && !failed; ++spins) {
        __builtin_ia32_pause();
        if (spins % 1024 != 0) continue;
        const clock::duration waited = clock::now() - start;
        if (waited < std::chrono::microseconds(500)) continue;
        check_stream();
        std::this_thread::sleep_for(std::min<clock::duration>(waited / 16, std::chrono::microseconds(500)));
        spins = 1023;  // (one look per sleep)
      }
    }
    auto take = [&](uint32_t i) {
      for (uint32_t spins = 1; __atomic_load_n(flags + i, __ATOMIC_ACQUIRE) != generation && !failed; ++spins) {
        __builtin_ia32_pause();
        if (spins % (1u << 16) == 0 && std::this_thread::get_id() == caller) check_stream();
      }
      if (failed) return;
      const size_t from = i * kPiece, len = n - from < kPiece ? n - from : kPiece;
      host_copy((uint8_t*)host + at + from, pipe.pinned + half * kHalf + from, len, bytes >= kPastCachesBytes);
    };
    if (stager.crew) {
      stager.crew->run(pieces, take, check_stream);
    } else {
      for (uint32_t i = 0; i < pieces; ++i) take(i);
    }
  }
  if (failed) {
    UK_HIP_OK(status);
    report_failure(__FILE__, __LINE__, __func__, "the copy to host memory ended without its flags");
    return false;
  }
  return true;
}

// Makes the operands of a call reachable from the device.
constexpr int kMostOperands = 10;
bool stage_operands(Stager& stager, Operand* const* ops, int count, hipStream_t stream) {
  Operand* mirrored[kMostOperands];
  int mirrors = 0, piped = 0;
  for (int i = 0; i < count; ++i) {
    Operand& o = *ops[i];
    o.dev = o.ptr;
    if (o.region.span == 0 || device_accessible(o.ptr)) continue;
    if (tl_async) {
      // Nothing is staged in asynchronous mode, and a host address must not
      // reach a kernel: the device would fault.
      report_failure(__FILE__, __LINE__, __func__, "asynchronous mode needs device-accessible operands");
      return false;
    }
    // (What is uploaded in one piece comes first.)
    if (o.upload && o.contiguous()) {
      for (int k = mirrors; k > piped; --k) mirrored[k] = mirrored[k - 1];
      mirrored[piped++] = &o;
    } else {
      mirrored[mirrors] = &o;
    }
    ++mirrors;
  }
  if (mirrors == 0) return true;
  // Whether the operands fit is settled before the first byte is copied.
  Checked need;
  int64_t total = 0;
  for (int i = 0; i < mirrors; ++i) total = need.add(total, need.add(mirrored[i]->region.span, 255) & ~(int64_t)255);
  if (!need.ok) {
    report_failure(__FILE__, __LINE__, __func__, stager.no_alloc
                       ? "host operands exceed IREE_UK_MI355X_NOALLOC_MAX_STAGED_BYTES of static staging memory"
                       : "host operands exceed the address space");
    return false;
  }
  uint8_t* base = nullptr;
  if (!stage_reserve(stager, (size_t)total, &base)) return false;
  size_t at = 0;
  for (int i = 0; i < mirrors; ++i) {
    Operand& o = *mirrored[i];
    o.host = o.ptr;
    o.dev = base + at;
    at += rounded_for_staging((size_t)o.region.span);
  }
  // The helpers are woken for what takes longer than waking them.
  if (stager.piped && total >= (int64_t)kPastCachesBytes && uk::HostCrew::instance().engage())
    stager.crew = &uk::HostCrew::instance();
  int i = 0;
  if (stager.piped && piped > 0) {
    stager.copies_issued = true;
    if (!pipe_up(stager, base, mirrored, piped, stream)) return false;
    i = piped;
  }
  for (; i < mirrors; ++i) {
    Operand& o = *mirrored[i];
    if (!o.upload) continue;
    stager.copies_issued = true;
    if (!copy_rows(const_cast<void*>(o.dev), o.host, o.region, hipMemcpyHostToDevice, stream)) return false;
  }
  return true;
}

bool finish(const Stager& stager, hipStream_t stream, const Operand& out) {
  if (out.host) {
    if (stager.piped && out.contiguous()) {
      if (pipe_down(stager, const_cast<void*>(out.host), out.dev, (size_t)out.region.span, stream)) return true;
      (void)hipStreamSynchronize(stream);
      return false;
    }
    if (!copy_rows(const_cast<void*>(out.host), out.dev, out.region, hipMemcpyDeviceToHost, stream)) {
      (void)hipStreamSynchronize(stream);
      return false;
    }
  }
  if (!tl_async) UK_HIP_OK(hipStreamSynchronize(stream));
  return true;
}

bool launch_ok(hipError_t e, const char* what) {
  if (e == hipSuccess) return true;
  char msg[256];
  snprintf(msg, sizeof msg, "%s launch -> %s", what, hipGetErrorString(e));
  report_failure(__FILE__, __LINE__, __func__, msg);
  return false;
}

// Leaves an entry point early after a failure: in synchronous mode nothing
// of the call may still be in flight when it returns (uploads read the
// caller's memory, and the staging memory is about to be handed on).
void abandon(const Stager& stager, hipStream_t stream) {
  if (!tl_async && stager.copies_issued) (void)hipStreamSynchronize(stream);
}

uk::Mmt4dLauncher select_mmt4d(const uk::Mmt4dArgs& a, bool probe_only) {
  uk::Mmt4dLauncher l = nullptr;
  if ((l = uk::select_mmt4d_gemv(a, probe_only))) return l;
  const uk::Mmt4dLauncher skinny = uk::select_mmt4d_skinny(a, probe_only);
  if (skinny && (probe_only || uk::mmt4d_skinny_preferred(a))) return skinny;
  if ((l = uk::select_mmt4d_mfma(a, probe_only))) return l;
  return skinny;
}

int pack_elem_bytes(uint32_t flags) {
  switch (flags & IREE_UK_FLAG_PACK_TYPE_MASK) {
    case IREE_UK_FLAG_PACK_TYPE_F32F32: return 4;
    case IREE_UK_FLAG_PACK_TYPE_I8I8: return 1;
    case IREE_UK_FLAG_PACK_TYPE_I32I32: return 4;
    case IREE_UK_FLAG_PACK_TYPE_F16F16: return 2;
    case IREE_UK_FLAG_PACK_TYPE_BF16BF16: return 2;
    default: return 0;
  }
}

int unpack_elem_bytes(uint32_t flags) {
  switch (flags & IREE_UK_FLAG_UNPACK_TYPE_MASK) {
    case IREE_UK_FLAG_UNPACK_TYPE_F32F32: return 4;
    case IREE_UK_FLAG_UNPACK_TYPE_I32I32: return 4;
    case IREE_UK_FLAG_UNPACK_TYPE_F16F16: return 2;
    case IREE_UK_FLAG_UNPACK_TYPE_BF16BF16: return 2;
    default: return 0;
  }
}

}  // namespace

//===----------------------------------------------------------------------===//
// mmt4d
//===----------------------------------------------------------------------===//

namespace {

void mmt4d_impl(const iree_uk_mmt4d_params_t* p, Stager& stager) {
  tl_last_kernel = "";
  UK_REQUIRE(p != nullptr);
  // Checks of mmt4d.c:12-48.
  const uint32_t known = IREE_UK_FLAG_MMT4D_TYPE_MASK | IREE_UK_FLAG_MMT4D_ACCUMULATE |
                         IREE_UK_FLAG_MMT4D_SKIP_INTERMEDIATE_ROUNDINGS |
                         IREE_UK_FLAG_MMT4D_ALLOW_GENERIC_FALLBACK_TILE_FUNCTION;
  UK_REQUIRE(!(p->flags & ~known));
  int lb = 0, rb = 0, ob = 0;
  UK_REQUIRE(uk::mmt4d_type_bits(p->flags, &lb, &rb, &ob));
  UK_REQUIRE(in_unsigned_range(p->M, 31));
  UK_REQUIRE(in_unsigned_range(p->N, 31));
  UK_REQUIRE(in_unsigned_range(p->K, 31));
  UK_REQUIRE(in_unsigned_range(p->M0, 15));
  UK_REQUIRE(in_unsigned_range(p->N0, 15));
  UK_REQUIRE(in_unsigned_range(p->K0, 15));
  UK_REQUIRE(ob >= 8);
  UK_REQUIRE((p->K0 * lb) % 8 == 0);
  UK_REQUIRE((p->K0 * rb) % 8 == 0);
  // (stride * bits) % 8 without forming the product.
  UK_REQUIRE(((p->lhs_stride0 % 8) * lb) % 8 == 0);
  UK_REQUIRE(((p->rhs_stride0 % 8) * rb) % 8 == 0);
  UK_REQUIRE(((p->lhs_offset % 8) * lb) % 8 == 0);
  UK_REQUIRE(((p->rhs_offset % 8) * rb) % 8 == 0);

  // Early exits of mmt4d.c:105-113. (K == 0 without ACCUMULATE still has to
  // zero the output tiles, so it goes on to a kernel.)
  const bool accumulate = p->flags & IREE_UK_FLAG_MMT4D_ACCUMULATE;
  if (p->M == 0 || p->N == 0 || (p->K == 0 && accumulate)) return;
  if (p->M0 == 0 || p->N0 == 0) return;  // empty tiles: nothing to write

  Checked c;
  const RowRegion lhs_region = make_region(c, p->M, c.bytes(c.mul(p->K, (int64_t)p->M0 * p->K0), lb),
                                           c.bytes(p->lhs_stride0, lb));
  const RowRegion rhs_region = make_region(c, p->N, c.bytes(c.mul(p->K, (int64_t)p->N0 * p->K0), rb),
                                           c.bytes(p->rhs_stride0, rb));
  const RowRegion out_region = make_region(c, p->M, c.bytes(c.mul(p->N, (int64_t)p->M0 * p->N0), ob),
                                           c.bytes(p->out_stride0, ob));
  const int64_t lhs_offset_bytes = c.bytes(p->lhs_offset, lb), rhs_offset_bytes = c.bytes(p->rhs_offset, rb),
                out_offset_bytes = c.bytes(p->out_offset, ob);
  UK_REQUIRE(c.ok && "operand extents fit int64");
  // The reference puts no condition on the strides (mmt4d.c:12-48). Operand
  // rows may overlap or coincide (stride 0 broadcasts one panel); they are
  // only read. Rows of the output may not overlap here, because they are
  // written concurrently, and strides that walk backwards are not supported.
  UK_REQUIRE(p->M == 1 || p->lhs_stride0 >= 0);
  UK_REQUIRE(p->N == 1 || p->rhs_stride0 >= 0);
  UK_REQUIRE(p->M == 1 || out_region.pitch >= out_region.width);

  const void* lhs = offset_pointer(p->lhs_buffer, lhs_offset_bytes);
  const void* rhs = offset_pointer(p->rhs_buffer, rhs_offset_bytes);
  const void* out = offset_pointer(p->out_buffer, out_offset_bytes);

  hipStream_t stream = tl_stream;
  // A host operand whose rows overlap is staged as one span.
  auto as_copied = [](const RowRegion& r) { return r.rows > 1 && r.pitch < r.width ? as_one_span(r) : r; };
  Operand o_lhs{lhs, as_copied(lhs_region), true}, o_rhs{rhs, as_copied(rhs_region), true}, o_out{out, out_region, accumulate};
  Operand* const operands[] = {&o_lhs, &o_rhs, &o_out};
  if (!stage_operands(stager, operands, 3, stream)) {
    abandon(stager, stream);
    return;
  }

  uk::Mmt4dArgs a;
  a.lhs = (const uint8_t*)o_lhs.dev;
  a.rhs = (const uint8_t*)o_rhs.dev;
  a.out = (uint8_t*)const_cast<void*>(o_out.dev);
  a.lhs_stride0 = p->lhs_stride0;
  a.rhs_stride0 = p->rhs_stride0;
  a.out_stride0 = p->out_stride0;
  a.M = p->M; a.N = p->N; a.K = p->K;
  a.M0 = p->M0; a.N0 = p->N0; a.K0 = p->K0;
  a.flags = p->flags;

  // The int4 kernels carry 16x the sums in int32, which holds for a total depth
  // below 131072. A deeper product is computed as a chain of calls over slices
  // of K, every slice after the first accumulating onto the output (exact:
  // int32 addition wraps the same way in any grouping).
  const int64_t depth_limit = 131072;
  if ((p->flags & IREE_UK_FLAG_MMT4D_TYPE_MASK) == IREE_UK_FLAG_MMT4D_TYPE_S8S4S32 && p->K0 > 0 &&
      p->K * p->K0 >= depth_limit && select_mmt4d(a, /*probe_only=*/true)) {
    // (A multiple of 8 k steps: whole 128-value steps of the matrix-vector kernel, whole chunks of the block kernels.)
    int64_t slice = (depth_limit - 1) / p->K0;
    if (slice > 8) slice &= ~(int64_t)7;
    for (int64_t k = 0; k < p->K; k += slice) {
      uk::Mmt4dArgs part = a;
      part.K = p->K - k < slice ? p->K - k : slice;
      part.lhs = a.lhs + k * p->M0 * p->K0;
      part.rhs = a.rhs + k * p->N0 * p->K0 / 2;
      if (k > 0) part.flags |= IREE_UK_FLAG_MMT4D_ACCUMULATE;
      uk::Mmt4dLauncher launcher = select_mmt4d(part, /*probe_only=*/false);
      if (!launcher) launcher = uk::launch_mmt4d_generic;
      if (!launch_ok(launcher(part, stream, &tl_last_kernel), "mmt4d")) {
        abandon(stager, stream);
        return;
      }
    }
    finish(stager, stream, o_out);
    return;
  }

  uk::Mmt4dLauncher launcher = select_mmt4d(a, /*probe_only=*/false);
  if (!launcher) launcher = uk::launch_mmt4d_generic;
  if (!launch_ok(launcher(a, stream, &tl_last_kernel), "mmt4d")) {
    abandon(stager, stream);
    return;
  }
  finish(stager, stream, o_out);
}

}  // namespace

UK_API void iree_uk_mmt4d_p(const iree_uk_mmt4d_params_t* p) {
  Stager stager;
  mmt4d_impl(p, stager);
}

UK_API void iree_uk_mi355x_mmt4d_noalloc_p(const iree_uk_mmt4d_params_t* p) {
  Stager stager;
  stager.no_alloc = true;
  mmt4d_impl(p, stager);
}

UK_API void iree_uk_mmt4d(const void* lhs_buffer, iree_uk_index_t lhs_offset,
                          iree_uk_index_t lhs_stride0, const void* rhs_buffer,
                          iree_uk_index_t rhs_offset, iree_uk_index_t rhs_stride0,
                          void* out_buffer, iree_uk_index_t out_offset, iree_uk_index_t out_stride0,
                          iree_uk_index_t M, iree_uk_index_t N, iree_uk_index_t K, int32_t M0,
                          int32_t N0, int32_t K0, uint32_t flags, const uint64_t* cpu_data) {
  iree_uk_mmt4d_params_t p;
  p.lhs_buffer = lhs_buffer; p.lhs_offset = lhs_offset; p.lhs_stride0 = lhs_stride0;
  p.rhs_buffer = rhs_buffer; p.rhs_offset = rhs_offset; p.rhs_stride0 = rhs_stride0;
  p.out_buffer = out_buffer; p.out_offset = out_offset; p.out_stride0 = out_stride0;
  p.M = M; p.N = N; p.K = K; p.M0 = M0; p.N0 = N0; p.K0 = K0;
  p.flags = flags; p.cpu_data = cpu_data;
  iree_uk_mmt4d_p(&p);
}

UK_API uint32_t iree_uk_mmt4d_info_p(const iree_uk_mmt4d_params_t* p) {
  if (!p) return 0;
  int lb, rb, ob;
  if (!uk::mmt4d_type_bits(p->flags, &lb, &rb, &ob)) return 0;
  uk::Mmt4dArgs a;
  memset(&a, 0, sizeof a);
  a.M0 = p->M0; a.N0 = p->N0; a.K0 = p->K0;
  a.flags = p->flags;
  return select_mmt4d(a, /*probe_only=*/true)
             ? IREE_UK_FLAG_MMT4D_INFO_HAVE_ARCHITECTURE_SPECIFIC_TILE_FUNCTION
             : 0u;
}

UK_API uint32_t iree_uk_mmt4d_info(int32_t M0, int32_t N0, int32_t K0, uint32_t flags,
                                   const uint64_t* cpu_data) {
  iree_uk_mmt4d_params_t p;
  memset(&p, 0, sizeof p);
  p.M0 = M0; p.N0 = N0; p.K0 = K0; p.flags = flags; p.cpu_data = cpu_data;
  return iree_uk_mmt4d_info_p(&p);
}

//===----------------------------------------------------------------------===//
// pack
//===----------------------------------------------------------------------===//

UK_API void iree_uk_pack_p(const iree_uk_pack_params_t* p) {
  tl_last_kernel = "";
  UK_REQUIRE(p != nullptr);
  // Checks of pack.c:51-103. The reference additionally limits one tile to its
  // 4 KiB stack buffer (pack.c:39-49); nothing here needs that limit.
  const uint32_t known = IREE_UK_FLAG_PACK_TRANSPOSE_INNER | IREE_UK_FLAG_PACK_TRANSPOSE_OUTER |
                         IREE_UK_FLAG_PACK_TYPE_MASK;
  UK_REQUIRE(!(p->flags & ~known));
  const int e = pack_elem_bytes(p->flags);
  UK_REQUIRE(e != 0);
  UK_REQUIRE(p->in_size0 >= 0);
  UK_REQUIRE(p->in_size1 >= 0);
  UK_REQUIRE(p->out_size0 >= 0);
  UK_REQUIRE(p->out_size1 >= 0);
  UK_REQUIRE(p->out_size2 >= 0);
  UK_REQUIRE(p->out_size3 >= 0);
  UK_REQUIRE(p->in_stride0 >= 0);
  UK_REQUIRE(p->in_stride1 >= 0);
  UK_REQUIRE(p->out_stride0 >= 0);
  Checked c;
  UK_REQUIRE(p->out_stride1 == c.mul(p->out_size2, p->out_size3) && c.ok);
  int64_t outer0 = p->out_size0, outer1 = p->out_size1;
  int64_t tile0 = p->out_size2, tile1 = p->out_size3;
  if (p->flags & IREE_UK_FLAG_PACK_TRANSPOSE_OUTER) { int64_t t = outer0; outer0 = outer1; outer1 = t; }
  if (p->flags & IREE_UK_FLAG_PACK_TRANSPOSE_INNER) { int64_t t = tile0; tile0 = tile1; tile1 = t; }
  UK_REQUIRE(tiles_cover(outer0, tile0, p->in_size0));
  UK_REQUIRE(tiles_cover(outer1, tile1, p->in_size1));

  // Early exit of pack.c:106-109.
  if (p->out_size0 == 0 || p->out_size1 == 0 || p->out_size2 == 0 || p->out_size3 == 0) return;

  const bool have_input = p->in_size0 > 0 && p->in_size1 > 0;
  const RowRegion in_region =
      make_region(c, have_input ? p->in_size0 : 0, c.mul(c.add(c.mul(p->in_size1 - 1, p->in_stride1), 1), e),
                  c.mul(p->in_stride0, e));
  const RowRegion out_region = make_region(
      c, p->out_size0, c.mul(c.mul(p->out_size1, p->out_stride1), e), c.mul(p->out_stride0, e));
  const int64_t in_offset_bytes = c.mul(p->in_offset, e), out_offset_bytes = c.mul(p->out_offset, e);
  UK_REQUIRE(c.ok && "operand extents fit int64");
  UK_REQUIRE(p->out_size0 == 1 || out_region.pitch >= out_region.width);

  const void* in = offset_pointer(p->in_buffer, in_offset_bytes);
  const void* out = offset_pointer(p->out_buffer, out_offset_bytes);

  hipStream_t stream = tl_stream;
  // A host input whose rows overlap or interleave (stride0 < row width) is
  // staged as one span.
  RowRegion in_copy = in_region;
  if (in_copy.rows > 1 && in_copy.pitch < in_copy.width) in_copy = as_one_span(in_region);
  Stager stager;
  Operand o_in{in, in_copy, true}, o_out{out, out_region, false};
  Operand* const operands[] = {&o_in, &o_out};
  if (!stage_operands(stager, operands, 2, stream)) {
    abandon(stager, stream);
    return;
  }

  uk::PackArgs a;
  a.in = (const uint8_t*)o_in.dev;
  a.out = (uint8_t*)const_cast<void*>(o_out.dev);
  a.in_stride0 = p->in_stride0; a.in_stride1 = p->in_stride1;
  a.out_stride0 = p->out_stride0;
  a.in_size0 = p->in_size0; a.in_size1 = p->in_size1;
  a.out_size0 = p->out_size0; a.out_size1 = p->out_size1;
  a.out_size2 = p->out_size2; a.out_size3 = p->out_size3;
  a.padding_value = p->padding_value;
  a.flags = p->flags;
  a.elem_bytes = e;
  if (!launch_ok(uk::launch_pack(a, stream, &tl_last_kernel), "pack")) {
    abandon(stager, stream);
    return;
  }
  finish(stager, stream, o_out);
}

UK_API void iree_uk_pack(const void* in_buffer, iree_uk_index_t in_offset, iree_uk_index_t in_stride0,
                         iree_uk_index_t in_stride1, void* out_buffer, iree_uk_index_t out_offset,
                         iree_uk_index_t out_stride0, iree_uk_index_t out_stride1,
                         iree_uk_index_t in_size0, iree_uk_index_t in_size1,
                         iree_uk_index_t out_size0, iree_uk_index_t out_size1,
                         iree_uk_index_t out_size2, iree_uk_index_t out_size3,
                         uint64_t padding_value, uint32_t flags, const uint64_t* cpu_data) {
  iree_uk_pack_params_t p;
  p.in_buffer = in_buffer; p.in_offset = in_offset;
  p.in_stride0 = in_stride0; p.in_stride1 = in_stride1;
  p.out_buffer = out_buffer; p.out_offset = out_offset;
  p.out_stride0 = out_stride0; p.out_stride1 = out_stride1;
  p.in_size0 = in_size0; p.in_size1 = in_size1;
  p.out_size0 = out_size0; p.out_size1 = out_size1;
  p.out_size2 = out_size2; p.out_size3 = out_size3;
  p.padding_value = padding_value; p.flags = flags; p.cpu_data = cpu_data;
  iree_uk_pack_p(&p);
}

//===----------------------------------------------------------------------===//
// unpack
//===----------------------------------------------------------------------===//

UK_API void iree_uk_unpack_p(const iree_uk_unpack_params_t* p) {
  tl_last_kernel = "";
  UK_REQUIRE(p != nullptr);
  // Checks of unpack.c:31-81 (tile-size limit of its stack buffer left out).
  const uint32_t known = IREE_UK_FLAG_UNPACK_TRANSPOSE_INNER |
                         IREE_UK_FLAG_UNPACK_TRANSPOSE_OUTER | IREE_UK_FLAG_UNPACK_TYPE_MASK;
  UK_REQUIRE(!(p->flags & ~known));
  const int e = unpack_elem_bytes(p->flags);
  UK_REQUIRE(e != 0);
  UK_REQUIRE(p->out_size0 >= 0);
  UK_REQUIRE(p->out_size1 >= 0);
  UK_REQUIRE(p->in_size0 >= 0);
  UK_REQUIRE(p->in_size1 >= 0);
  UK_REQUIRE(p->in_size2 >= 0);
  UK_REQUIRE(p->in_size3 >= 0);
  UK_REQUIRE(p->in_stride0 >= 0);
  Checked c;
  UK_REQUIRE(p->in_stride1 == c.mul(p->in_size2, p->in_size3) && c.ok);
  UK_REQUIRE(p->out_stride0 >= 0);
  UK_REQUIRE(p->out_stride1 >= 0);
  int64_t outer0 = p->in_size0, outer1 = p->in_size1;
  int64_t tile0 = p->in_size2, tile1 = p->in_size3;
  if (p->flags & IREE_UK_FLAG_UNPACK_TRANSPOSE_OUTER) { int64_t t = outer0; outer0 = outer1; outer1 = t; }
  if (p->flags & IREE_UK_FLAG_UNPACK_TRANSPOSE_INNER) { int64_t t = tile0; tile0 = tile1; tile1 = t; }
  UK_REQUIRE(tiles_cover(outer0, tile0, p->out_size0));
  UK_REQUIRE(tiles_cover(outer1, tile1, p->out_size1));

  // Early exit of unpack.c:84-86.
  if (p->out_size0 == 0 || p->out_size1 == 0) return;

  const RowRegion in_region =
      make_region(c, p->in_size0, c.mul(c.mul(p->in_size1, p->in_stride1), e), c.mul(p->in_stride0, e));
  const RowRegion out_region =
      make_region(c, p->out_size0, c.mul(c.add(c.mul(p->out_size1 - 1, p->out_stride1), 1), e),
                  c.mul(p->out_stride0, e));
  const int64_t in_offset_bytes = c.mul(p->in_offset, e), out_offset_bytes = c.mul(p->out_offset, e);
  UK_REQUIRE(c.ok && "operand extents fit int64");
  UK_REQUIRE(p->in_size0 == 1 || in_region.pitch >= in_region.width);
  UK_REQUIRE(p->out_size0 == 1 || out_region.pitch >= out_region.width);

  const void* in = offset_pointer(p->in_buffer, in_offset_bytes);
  const void* out = offset_pointer(p->out_buffer, out_offset_bytes);

  hipStream_t stream = tl_stream;
  Stager stager;
  // With an inner output stride the bytes between elements must survive the
  // round trip through the staging buffer, so the rows are uploaded first.
  Operand o_in{in, in_region, true}, o_out{out, out_region, p->out_stride1 != 1};
  Operand* const operands[] = {&o_in, &o_out};
  if (!stage_operands(stager, operands, 2, stream)) {
    abandon(stager, stream);
    return;
  }

  uk::UnpackArgs a;
  a.in = (const uint8_t*)o_in.dev;
  a.out = (uint8_t*)const_cast<void*>(o_out.dev);
  a.in_stride0 = p->in_stride0;
  a.out_stride0 = p->out_stride0; a.out_stride1 = p->out_stride1;
  a.in_size0 = p->in_size0; a.in_size1 = p->in_size1;
  a.in_size2 = p->in_size2; a.in_size3 = p->in_size3;
  a.out_size0 = p->out_size0; a.out_size1 = p->out_size1;
  a.flags = p->flags;
  a.elem_bytes = e;
  if (!launch_ok(uk::launch_unpack(a, stream, &tl_last_kernel), "unpack")) {
    abandon(stager, stream);
    return;
  }
  finish(stager, stream, o_out);
}

UK_API void iree_uk_unpack(const void* in_buffer, iree_uk_index_t in_offset,
                           iree_uk_index_t in_stride0, iree_uk_index_t in_stride1, void* out_buffer,
                           iree_uk_index_t out_offset, iree_uk_index_t out_stride0,
                           iree_uk_index_t out_stride1, iree_uk_index_t in_size0,
                           iree_uk_index_t in_size1, iree_uk_index_t in_size2,
                           iree_uk_index_t in_size3, iree_uk_index_t out_size0,
                           iree_uk_index_t out_size1, uint32_t flags, const uint64_t* cpu_data) {
  iree_uk_unpack_params_t p;
  p.in_buffer = in_buffer; p.in_offset = in_offset;
  p.in_stride0 = in_stride0; p.in_stride1 = in_stride1;
  p.out_buffer = out_buffer; p.out_offset = out_offset;
  p.out_stride0 = out_stride0; p.out_stride1 = out_stride1;
  p.in_size0 = in_size0; p.in_size1 = in_size1; p.in_size2 = in_size2; p.in_size3 = in_size3;
  p.out_size0 = out_size0; p.out_size1 = out_size1;
  p.flags = flags; p.cpu_data = cpu_data;
  iree_uk_unpack_p(&p);
}

//===----------------------------------------------------------------------===//
// query_tile_sizes
//===----------------------------------------------------------------------===//

UK_API void iree_uk_query_tile_sizes_2d(const iree_uk_query_tile_sizes_2d_params_t* p,
                                        iree_uk_query_tile_sizes_2d_out_params_t* o) {
  UK_REQUIRE(p != nullptr && o != nullptr);
  // Tile shapes whose mmt4d runs on an MFMA kernel of this library: one
  // 16x16 MFMA output block per tile, K0 = the bytes one lane feeds per MFMA.
  int M0 = 16, N0 = 16, K0 = 0;
  switch (p->flags & IREE_UK_FLAG_QUERY_TILE_SIZES_OPERATION_MASK) {
    case IREE_UK_FLAG_QUERY_TILE_SIZES_OPERATION_MATMUL_I8I8I32: K0 = 64; break;
    case IREE_UK_FLAG_QUERY_TILE_SIZES_OPERATION_MATMUL_F16F16F32:
    case IREE_UK_FLAG_QUERY_TILE_SIZES_OPERATION_MATMUL_F16F16F16:
    case IREE_UK_FLAG_QUERY_TILE_SIZES_OPERATION_MATMUL_BF16BF16F32:
    case IREE_UK_FLAG_QUERY_TILE_SIZES_OPERATION_MATMUL_BF16BF16BF16: K0 = 16; break;
    case IREE_UK_FLAG_QUERY_TILE_SIZES_OPERATION_MATMUL_F32F32F32: K0 = 4; break;
    default: break;
  }
  UK_REQUIRE(K0 != 0);
  switch (p->flags & IREE_UK_FLAG_QUERY_TILE_SIZES_OPERAND_ROLE_MASK) {
    case IREE_UK_FLAG_QUERY_TILE_SIZES_OPERAND_ROLE_LHS: o->tile_size0 = M0; o->tile_size1 = K0; break;
    case IREE_UK_FLAG_QUERY_TILE_SIZES_OPERAND_ROLE_RHS: o->tile_size0 = N0; o->tile_size1 = K0; break;
    case IREE_UK_FLAG_QUERY_TILE_SIZES_OPERAND_ROLE_RESULT: o->tile_size0 = M0; o->tile_size1 = N0; break;
    default: UK_REQUIRE(!"unknown operand role");
  }
}

//===----------------------------------------------------------------------===//
// Microscaled operators and the norm (no counterpart in the reference)
//===----------------------------------------------------------------------===//

namespace {

// Whether an operand that is written shares bytes with another one. Rows that interleave at the same pitch (column ranges
// of one wider matrix) do not; any other two spans that cross are taken to.
bool overlap(const Operand& a, const Operand& b) {
  if (a.region.span == 0 || b.region.span == 0) return false;
  const uintptr_t x = (uintptr_t)a.ptr, y = (uintptr_t)b.ptr;
  if (x + (uintptr_t)a.region.span <= y || y + (uintptr_t)b.region.span <= x) return false;
  const int64_t pitch = a.region.pitch;
  if (pitch != b.region.pitch || a.region.rows == 1 || b.region.rows == 1) return true;
  const int64_t between = x <= y ? (int64_t)((y - x) % (uintptr_t)pitch) : (pitch - (int64_t)((x - y) % (uintptr_t)pitch)) % pitch;
  return between < a.region.width || between + b.region.width > pitch;
}

// Whether an operand that a call touches has a buffer.
bool given(const Operand& o, const void* buffer) { return o.region.span == 0 || buffer != nullptr; }

bool same_place(const Operand& a, const Operand& b) {
  return a.ptr == b.ptr && (a.region.rows == 1 || a.region.pitch == b.region.pitch);
}

// Rows that are written concurrently lie apart.
bool rows_apart(const RowRegion& r) { return r.rows <= 1 || r.pitch >= r.width; }

RowRegion as_copied(const RowRegion& r) { return r.rows > 1 && r.pitch < r.width ? as_one_span(r) : r; }

// Ends a call with several results: every one of them back where the caller has it.
bool finish(const Stager& stager, hipStream_t stream, const Operand* const* outs, int count) {
  for (int i = 0; i < count; ++i) {
    if (outs[i]->host && !finish(stager, stream, *outs[i])) return false;
  }
  if (!tl_async) UK_HIP_OK(hipStreamSynchronize(stream));
  return true;
}

// Type flags of these operators number the float types 1 to 3, once for each other type of the call.
uk::Float float_of(uint32_t type) { return (uk::Float)((type - 1) % 3); }

}  // namespace

UK_API void iree_uk_mi355x_mx_pack_p(const iree_uk_mi355x_mx_pack_params_t* p) {
  tl_last_kernel = "";
  UK_REQUIRE(p != nullptr);
  UK_REQUIRE(!(p->flags & ~(uint32_t)IREE_UK_MI355X_FLAG_MX_PACK_TYPE_MASK));
  UK_REQUIRE(p->flags >= IREE_UK_MI355X_FLAG_MX_PACK_TYPE_F32E2M1 &&
             p->flags <= IREE_UK_MI355X_FLAG_MX_PACK_TYPE_BF16E4M3);
  const uk::Float type = float_of(p->flags);
  const int e = uk::float_bytes(type), bits = p->flags <= IREE_UK_MI355X_FLAG_MX_PACK_TYPE_BF16E2M1 ? 4 : 8;
  UK_REQUIRE(p->in_size0 >= 0);
  UK_REQUIRE(p->in_size1 >= 0);
  UK_REQUIRE(p->out_size0 >= 0);
  UK_REQUIRE(p->out_size1 >= 0);
  UK_REQUIRE(p->out_size2 >= 0);
  UK_REQUIRE(p->out_size3 >= 0);
  UK_REQUIRE(p->in_stride0 >= 0);
  UK_REQUIRE(p->in_stride1 >= 0);
  UK_REQUIRE(p->out_stride0 >= 0);
  UK_REQUIRE(p->scales_stride0 >= 0);
  UK_REQUIRE(p->out_size3 % 32 == 0);
  UK_REQUIRE(bits == 8 || (p->out_offset % 2 == 0 && p->out_stride0 % 2 == 0));
  UK_REQUIRE(tiles_cover(p->out_size0, p->out_size2, p->in_size0));
  UK_REQUIRE(tiles_cover(p->out_size1, p->out_size3, p->in_size1));
  if (p->out_size0 == 0 || p->out_size1 == 0 || p->out_size2 == 0 || p->out_size3 == 0) return;

  Checked c;
  const bool have_input = p->in_size0 > 0 && p->in_size1 > 0;
  const RowRegion in_region =
      make_region(c, have_input ? p->in_size0 : 0, c.mul(c.add(c.mul(p->in_size1 - 1, p->in_stride1), 1), e),
                  c.mul(p->in_stride0, e));
  const int64_t row = c.mul(p->out_size1, c.mul(p->out_size2, p->out_size3));
  const RowRegion codes_region = make_region(c, p->out_size0, c.bytes(row, bits), c.bytes(p->out_stride0, bits));
  const RowRegion scales_region = make_region(c, p->out_size0, row / 32, p->scales_stride0);
  const int64_t in_offset_bytes = c.mul(p->in_offset, e), out_offset_bytes = c.bytes(p->out_offset, bits);
  UK_REQUIRE(c.ok && "operand extents fit int64");
  UK_REQUIRE(rows_apart(codes_region));
  UK_REQUIRE(rows_apart(scales_region));

  hipStream_t stream = tl_stream;
  Stager stager;
  Operand o_in{offset_pointer(p->in_buffer, in_offset_bytes), as_copied(in_region), true};
  Operand o_codes{offset_pointer(p->out_buffer, out_offset_bytes), codes_region, false};
  Operand o_scales{offset_pointer(p->scales_buffer, p->scales_offset), scales_region, false};
  UK_REQUIRE(!overlap(o_codes, o_scales));
  UK_REQUIRE(!overlap(o_codes, o_in));
  UK_REQUIRE(!overlap(o_scales, o_in));
  Operand* const operands[] = {&o_in, &o_codes, &o_scales};
  UK_REQUIRE(given(o_in, p->in_buffer));
  UK_REQUIRE(given(o_codes, p->out_buffer));
  UK_REQUIRE(given(o_scales, p->scales_buffer));
  if (!stage_operands(stager, operands, 3, stream)) {
    abandon(stager, stream);
    return;
  }
  uk::MxPackArgs a;
  a.in = (const uint8_t*)o_in.dev;
  a.codes = (uint8_t*)const_cast<void*>(o_codes.dev);
  a.scales = (uint8_t*)const_cast<void*>(o_scales.dev);
  a.in_stride0 = p->in_stride0; a.in_stride1 = p->in_stride1;
  a.codes_stride0 = codes_region.pitch; a.scales_stride0 = scales_region.pitch;
  a.in_size0 = p->in_size0; a.in_size1 = p->in_size1;
  a.outer0 = p->out_size0; a.outer1 = p->out_size1; a.tile0 = p->out_size2; a.tile1 = p->out_size3;
  a.type = type;
  a.bits = bits;
  if (!launch_ok(uk::launch_mx_pack(a, stream, &tl_last_kernel), "mx_pack")) {
    abandon(stager, stream);
    return;
  }
  const Operand* const outs[] = {&o_codes, &o_scales};
  finish(stager, stream, outs, 2);
}

UK_API void iree_uk_mi355x_mx_unpack_p(const iree_uk_mi355x_mx_unpack_params_t* p) {
  tl_last_kernel = "";
  UK_REQUIRE(p != nullptr);
  UK_REQUIRE(!(p->flags & ~(uint32_t)IREE_UK_MI355X_FLAG_MX_UNPACK_TYPE_MASK));
  UK_REQUIRE(p->flags >= IREE_UK_MI355X_FLAG_MX_UNPACK_TYPE_E2M1F32 &&
             p->flags <= IREE_UK_MI355X_FLAG_MX_UNPACK_TYPE_E4M3BF16);
  const uk::Float type = float_of(p->flags);
  const int e = uk::float_bytes(type), bits = p->flags <= IREE_UK_MI355X_FLAG_MX_UNPACK_TYPE_E2M1BF16 ? 4 : 8;
  UK_REQUIRE(p->out_size0 >= 0);
  UK_REQUIRE(p->out_size1 >= 0);
  UK_REQUIRE(p->in_size0 >= 0);
  UK_REQUIRE(p->in_size1 >= 0);
  UK_REQUIRE(p->in_size2 >= 0);
  UK_REQUIRE(p->in_size3 >= 0);
  UK_REQUIRE(p->in_stride0 >= 0);
  UK_REQUIRE(p->scales_stride0 >= 0);
  UK_REQUIRE(p->out_stride0 >= 0);
  UK_REQUIRE(p->out_stride1 >= 0);
  UK_REQUIRE(p->in_size3 % 32 == 0);
  UK_REQUIRE(bits == 8 || (p->in_offset % 2 == 0 && p->in_stride0 % 2 == 0));
  UK_REQUIRE(tiles_cover(p->in_size0, p->in_size2, p->out_size0));
  UK_REQUIRE(tiles_cover(p->in_size1, p->in_size3, p->out_size1));
  if (p->out_size0 == 0 || p->out_size1 == 0) return;

  Checked c;
  const int64_t row = c.mul(p->in_size1, c.mul(p->in_size2, p->in_size3));
  const RowRegion codes_region = make_region(c, p->in_size0, c.bytes(row, bits), c.bytes(p->in_stride0, bits));
  const RowRegion scales_region = make_region(c, p->in_size0, row / 32, p->scales_stride0);
  const RowRegion out_region =
      make_region(c, p->out_size0, c.mul(c.add(c.mul(p->out_size1 - 1, p->out_stride1), 1), e), c.mul(p->out_stride0, e));
  const int64_t in_offset_bytes = c.bytes(p->in_offset, bits), out_offset_bytes = c.mul(p->out_offset, e);
  UK_REQUIRE(c.ok && "operand extents fit int64");
  UK_REQUIRE(rows_apart(out_region));
  UK_REQUIRE(p->out_size1 == 1 || p->out_stride1 >= 1);

  hipStream_t stream = tl_stream;
  Stager stager;
  Operand o_codes{offset_pointer(p->in_buffer, in_offset_bytes), as_copied(codes_region), true};
  Operand o_scales{offset_pointer(p->scales_buffer, p->scales_offset), as_copied(scales_region), true};
  // (With an inner stride the bytes between elements have to survive the way through the staging memory.)
  Operand o_out{offset_pointer(p->out_buffer, out_offset_bytes), out_region, p->out_stride1 != 1};
  UK_REQUIRE(!overlap(o_out, o_codes));
  UK_REQUIRE(!overlap(o_out, o_scales));
  Operand* const operands[] = {&o_codes, &o_scales, &o_out};
  UK_REQUIRE(given(o_codes, p->in_buffer));
  UK_REQUIRE(given(o_scales, p->scales_buffer));
  UK_REQUIRE(given(o_out, p->out_buffer));
  if (!stage_operands(stager, operands, 3, stream)) {
    abandon(stager, stream);
    return;
  }
  uk::MxUnpackArgs a;
  a.codes = (const uint8_t*)o_codes.dev;
  a.scales = (const uint8_t*)o_scales.dev;
  a.out = (uint8_t*)const_cast<void*>(o_out.dev);
  a.codes_stride0 = codes_region.pitch; a.scales_stride0 = scales_region.pitch;
  a.out_stride0 = p->out_stride0; a.out_stride1 = p->out_stride1;
  a.outer0 = p->in_size0; a.outer1 = p->in_size1; a.tile0 = p->in_size2; a.tile1 = p->in_size3;
  a.out_size0 = p->out_size0; a.out_size1 = p->out_size1;
  a.type = type;
  a.bits = bits;
  if (!launch_ok(uk::launch_mx_unpack(a, stream, &tl_last_kernel), "mx_unpack")) {
    abandon(stager, stream);
    return;
  }
  finish(stager, stream, o_out);
}

UK_API void iree_uk_mi355x_mx_mmt4d_p(const iree_uk_mi355x_mx_mmt4d_params_t* p) {
  tl_last_kernel = "";
  UK_REQUIRE(p != nullptr);
  const uint32_t known = IREE_UK_MI355X_FLAG_MX_MMT4D_TYPE_MASK | IREE_UK_MI355X_FLAG_MX_MMT4D_ACCUMULATE;
  UK_REQUIRE(!(p->flags & ~known));
  const uint32_t type = p->flags & IREE_UK_MI355X_FLAG_MX_MMT4D_TYPE_MASK;
  UK_REQUIRE(type >= IREE_UK_MI355X_FLAG_MX_MMT4D_TYPE_E2M1E2M1F32 &&
             type <= IREE_UK_MI355X_FLAG_MX_MMT4D_TYPE_E4M3E2M1BF16);
  const int lb = type <= IREE_UK_MI355X_FLAG_MX_MMT4D_TYPE_E2M1E2M1BF16 ? 4 : 8;
  const uk::Float out_type = float_of(type);
  const int e = uk::float_bytes(out_type);
  UK_REQUIRE(in_unsigned_range(p->M, 31));
  UK_REQUIRE(in_unsigned_range(p->N, 31));
  UK_REQUIRE(in_unsigned_range(p->K, 31));
  UK_REQUIRE(in_unsigned_range(p->M0, 15));
  UK_REQUIRE(in_unsigned_range(p->N0, 15));
  UK_REQUIRE(in_unsigned_range(p->K0, 15));
  UK_REQUIRE(p->K0 % 32 == 0);
  UK_REQUIRE(lb == 8 || (p->lhs_offset % 2 == 0 && p->lhs_stride0 % 2 == 0));
  UK_REQUIRE(p->rhs_offset % 2 == 0 && p->rhs_stride0 % 2 == 0);
  const bool accumulate = p->flags & IREE_UK_MI355X_FLAG_MX_MMT4D_ACCUMULATE;
  if (p->M == 0 || p->N == 0 || ((p->K == 0 || p->K0 == 0) && accumulate)) return;
  if (p->M0 == 0 || p->N0 == 0) return;

  Checked c;
  const int64_t lhs_row = c.mul(p->K, (int64_t)p->M0 * p->K0), rhs_row = c.mul(p->K, (int64_t)p->N0 * p->K0);
  const RowRegion lhs_region = make_region(c, p->M, c.bytes(lhs_row, lb), c.bytes(p->lhs_stride0, lb));
  const RowRegion rhs_region = make_region(c, p->N, c.bytes(rhs_row, 4), c.bytes(p->rhs_stride0, 4));
  const RowRegion lhs_scales_region = make_region(c, p->M, lhs_row / 32, p->lhs_scales_stride0);
  const RowRegion rhs_scales_region = make_region(c, p->N, rhs_row / 32, p->rhs_scales_stride0);
  const RowRegion out_region =
      make_region(c, p->M, c.mul(c.mul(p->N, (int64_t)p->M0 * p->N0), e), c.mul(p->out_stride0, e));
  const int64_t lhs_offset_bytes = c.bytes(p->lhs_offset, lb), rhs_offset_bytes = c.bytes(p->rhs_offset, 4),
                out_offset_bytes = c.mul(p->out_offset, e);
  UK_REQUIRE(c.ok && "operand extents fit int64");
  // Panels of the operands may coincide or overlap (they are only read); see iree_uk_mmt4d.
  UK_REQUIRE(p->M == 1 || (p->lhs_stride0 >= 0 && p->lhs_scales_stride0 >= 0));
  UK_REQUIRE(p->N == 1 || (p->rhs_stride0 >= 0 && p->rhs_scales_stride0 >= 0));
  UK_REQUIRE(rows_apart(out_region));

  hipStream_t stream = tl_stream;
  Stager stager;
  Operand o_lhs{offset_pointer(p->lhs_buffer, lhs_offset_bytes), as_copied(lhs_region), true};
  Operand o_lhs_scales{offset_pointer(p->lhs_scales_buffer, p->lhs_scales_offset), as_copied(lhs_scales_region), true};
  Operand o_rhs{offset_pointer(p->rhs_buffer, rhs_offset_bytes), as_copied(rhs_region), true};
  Operand o_rhs_scales{offset_pointer(p->rhs_scales_buffer, p->rhs_scales_offset), as_copied(rhs_scales_region), true};
  Operand o_out{offset_pointer(p->out_buffer, out_offset_bytes), out_region, accumulate};
  Operand* const operands[] = {&o_lhs, &o_lhs_scales, &o_rhs, &o_rhs_scales, &o_out};
  UK_REQUIRE(given(o_lhs, p->lhs_buffer));
  UK_REQUIRE(given(o_lhs_scales, p->lhs_scales_buffer));
  UK_REQUIRE(given(o_rhs, p->rhs_buffer));
  UK_REQUIRE(given(o_rhs_scales, p->rhs_scales_buffer));
  UK_REQUIRE(given(o_out, p->out_buffer));
  for (int i = 0; i < 4; ++i) UK_REQUIRE(!overlap(o_out, *operands[i]));
  if (!stage_operands(stager, operands, 5, stream)) {
    abandon(stager, stream);
    return;
  }
  uk::MxMmt4dArgs a;
  a.lhs = (const uint8_t*)o_lhs.dev;
  a.lhs_scales = (const uint8_t*)o_lhs_scales.dev;
  a.rhs = (const uint8_t*)o_rhs.dev;
  a.rhs_scales = (const uint8_t*)o_rhs_scales.dev;
  a.out = (uint8_t*)const_cast<void*>(o_out.dev);
  a.lhs_stride0 = lhs_region.pitch; a.lhs_scales_stride0 = lhs_scales_region.pitch;
  a.rhs_stride0 = rhs_region.pitch; a.rhs_scales_stride0 = rhs_scales_region.pitch;
  a.out_stride0 = p->out_stride0;
  a.M = p->M; a.N = p->N; a.K = p->K0 == 0 ? 0 : p->K;
  a.M0 = p->M0; a.N0 = p->N0; a.K0 = p->K0 == 0 ? 32 : p->K0;
  a.lhs_bits = lb;
  a.out_type = out_type;
  a.accumulate = accumulate;
  if (!launch_ok(uk::launch_mx_mmt4d(a, stream, &tl_last_kernel), "mx_mmt4d")) {
    abandon(stager, stream);
    return;
  }
  finish(stager, stream, o_out);
}

UK_API void iree_uk_mi355x_rms_norm_p(const iree_uk_mi355x_rms_norm_params_t* p) {
  tl_last_kernel = "";
  UK_REQUIRE(p != nullptr);
  const uint32_t known = IREE_UK_MI355X_FLAG_RMS_NORM_TYPE_MASK | IREE_UK_MI355X_FLAG_RMS_NORM_WEIGHT_F32;
  UK_REQUIRE(!(p->flags & ~known));
  const uint32_t flag = p->flags & IREE_UK_MI355X_FLAG_RMS_NORM_TYPE_MASK;
  UK_REQUIRE(flag >= IREE_UK_MI355X_FLAG_RMS_NORM_TYPE_F32S8 && flag <= IREE_UK_MI355X_FLAG_RMS_NORM_TYPE_BF16E2M1);
  const uk::Float type = float_of(flag);
  const uk::NormOut out_type = (uk::NormOut)((flag - 1) / 3);
  const uk::Float weight_type = p->flags & IREE_UK_MI355X_FLAG_RMS_NORM_WEIGHT_F32 ? uk::Float::kF32 : type;
  const int e = uk::float_bytes(type), bits = out_type == uk::NormOut::kE2M1 ? 4 : 8;
  const bool rows_of_bytes = out_type != uk::NormOut::kS8;  // scales: bytes in rows, or one f32 a row
  UK_REQUIRE(p->size0 >= 0);
  UK_REQUIRE(p->size1 >= 0);
  UK_REQUIRE(p->out_size1 >= p->size1);
  UK_REQUIRE(!rows_of_bytes || p->out_size1 % 32 == 0);
  UK_REQUIRE(p->in_stride0 >= 0);
  UK_REQUIRE(!p->residual_buffer || p->residual_stride0 >= 0);
  UK_REQUIRE(!p->sum_buffer || (p->residual_buffer && p->sum_stride0 >= 0));
  UK_REQUIRE(p->out_stride0 >= 0);
  UK_REQUIRE(p->scales_stride0 >= 0);
  UK_REQUIRE(p->epsilon >= 0);
  UK_REQUIRE(bits == 8 || (p->out_offset % 2 == 0 && p->out_stride0 % 2 == 0));
  if (p->size0 == 0 || p->out_size1 == 0) return;

  Checked c;
  const int64_t width = c.mul(p->size1, e);
  const RowRegion in_region = make_region(c, p->size0, width, c.mul(p->in_stride0, e));
  const RowRegion residual_region =
      make_region(c, p->residual_buffer ? p->size0 : 0, width, c.mul(p->residual_buffer ? p->residual_stride0 : 0, e));
  const RowRegion sum_region =
      make_region(c, p->sum_buffer ? p->size0 : 0, width, c.mul(p->sum_buffer ? p->sum_stride0 : 0, e));
  const int weight_bytes = uk::float_bytes(weight_type);
  const RowRegion weight_region = make_region(c, p->weight_buffer ? 1 : 0, c.mul(p->size1, weight_bytes), 0);
  const RowRegion out_region = make_region(c, p->size0, c.bytes(p->out_size1, bits),
                                            c.bytes(p->out_stride0, bits));
  const int scale_bytes = rows_of_bytes ? 1 : 4;
  const RowRegion scales_region =
      make_region(c, p->size0, rows_of_bytes ? p->out_size1 / 32 : 4, c.mul(p->scales_stride0, scale_bytes));
  const int64_t in_offset = c.mul(p->in_offset, e), residual_offset = c.mul(p->residual_buffer ? p->residual_offset : 0, e),
                sum_offset = c.mul(p->sum_buffer ? p->sum_offset : 0, e),
                weight_offset = c.mul(p->weight_buffer ? p->weight_offset : 0, weight_bytes),
                out_offset = c.bytes(p->out_offset, bits), scales_offset = c.mul(p->scales_offset, scale_bytes);
  UK_REQUIRE(c.ok && "operand extents fit int64");
  UK_REQUIRE(rows_apart(sum_region));
  UK_REQUIRE(rows_apart(out_region));
  UK_REQUIRE(rows_apart(scales_region));

  hipStream_t stream = tl_stream;
  Stager stager;
  Operand o_in{offset_pointer(p->in_buffer, in_offset), as_copied(in_region), true};
  Operand o_residual{offset_pointer(p->residual_buffer, residual_offset), as_copied(residual_region), true};
  Operand o_sum{offset_pointer(p->sum_buffer, sum_offset), sum_region, false};
  Operand o_weight{offset_pointer(p->weight_buffer, weight_offset), weight_region, true};
  Operand o_out{offset_pointer(p->out_buffer, out_offset), out_region, false};
  Operand o_scales{offset_pointer(p->scales_buffer, scales_offset), scales_region, false};
  UK_REQUIRE(same_place(o_sum, o_in) || !overlap(o_sum, o_in));
  UK_REQUIRE(same_place(o_sum, o_residual) || !overlap(o_sum, o_residual));
  UK_REQUIRE(!overlap(o_sum, o_weight));
  const Operand* const inputs[] = {&o_in, &o_residual, &o_sum, &o_weight};
  for (const Operand* i : inputs) {
    UK_REQUIRE(!overlap(o_out, *i));
    UK_REQUIRE(!overlap(o_scales, *i));
  }
  UK_REQUIRE(!overlap(o_out, o_scales));
  Operand* const operands[] = {&o_in, &o_residual, &o_sum, &o_weight, &o_out, &o_scales};
  UK_REQUIRE(given(o_in, p->in_buffer));
  UK_REQUIRE(given(o_out, p->out_buffer));
  UK_REQUIRE(given(o_scales, p->scales_buffer));
  if (!stage_operands(stager, operands, 6, stream)) {
    abandon(stager, stream);
    return;
  }
  uk::RmsNormArgs a;
  a.in = (const uint8_t*)o_in.dev;
  a.residual = p->residual_buffer ? (const uint8_t*)o_residual.dev : nullptr;
  a.sum = p->sum_buffer ? (uint8_t*)const_cast<void*>(o_sum.dev) : nullptr;
  a.weight = p->weight_buffer ? (const uint8_t*)o_weight.dev : nullptr;
  a.out = (uint8_t*)const_cast<void*>(o_out.dev);
  a.scales = (uint8_t*)const_cast<void*>(o_scales.dev);
  a.in_stride0 = p->in_stride0; a.residual_stride0 = p->residual_stride0; a.sum_stride0 = p->sum_stride0;
  a.out_stride0 = out_region.pitch; a.scales_stride0 = scales_region.pitch;
  a.size0 = p->size0; a.size1 = p->size1; a.out_size1 = p->out_size1;
  a.epsilon = p->epsilon;
  a.type = type; a.weight_type = weight_type; a.out_type = out_type; a.stream_sum = false;
  if (!launch_ok(uk::launch_rms_norm(a, stream, &tl_last_kernel), "rms_norm")) {
    abandon(stager, stream);
    return;
  }
  const Operand* const outs[] = {&o_sum, &o_out, &o_scales};
  finish(stager, stream, outs, 3);
}

//===----------------------------------------------------------------------===//
// Feed-forward operators (no counterpart in the reference)
//===----------------------------------------------------------------------===//

namespace {

// Type flags number the operands' types 1 and 3, with an f32 result, and 2 and 4, with a result of the operands' type.
uk::Float operand_type_of(uint32_t type) { return type <= 2 ? uk::Float::kF16 : uk::Float::kBf16; }
uk::Float result_type_of(uint32_t type) { return type % 2 ? uk::Float::kF32 : operand_type_of(type); }

bool tile_counts_in_range(int64_t M, int64_t N, int64_t K, int32_t M0, int32_t N0, int32_t K0) {
  return in_unsigned_range(M, 31) && in_unsigned_range(N, 31) && in_unsigned_range(K, 31) && in_unsigned_range(M0, 15) &&
         in_unsigned_range(N0, 15) && in_unsigned_range(K0, 15);
}

constexpr uint32_t kGatedKnown = IREE_UK_MI355X_FLAG_GATED_MMT4D_TYPE_MASK |
                                 IREE_UK_MI355X_FLAG_GATED_MMT4D_ACTIVATION_MASK | IREE_UK_MI355X_FLAG_GATED_MMT4D_PRE_F32;
bool gated_flags_known(uint32_t flags, uint32_t more) {
  const uint32_t type = flags & IREE_UK_MI355X_FLAG_GATED_MMT4D_TYPE_MASK;
  const uint32_t activation = flags & IREE_UK_MI355X_FLAG_GATED_MMT4D_ACTIVATION_MASK;
  return !(flags & ~(kGatedKnown | more)) && type >= IREE_UK_MI355X_FLAG_GATED_MMT4D_TYPE_F16F16F32 &&
         type <= IREE_UK_MI355X_FLAG_GATED_MMT4D_TYPE_BF16BF16BF16 && activation >= IREE_UK_MI355X_FLAG_GATED_MMT4D_SILU &&
         activation <= IREE_UK_MI355X_FLAG_GATED_MMT4D_SIGMOID;
}
uk::Activation activation_of(uint32_t flags) {
  return (uk::Activation)(((flags & IREE_UK_MI355X_FLAG_GATED_MMT4D_ACTIVATION_MASK) >> 8) - 1);
}

// A tiled operand [outer0][outer1][tile0][tile1] of `bytes` an element (outer0 = 0: none).
RowRegion tiled_region(Checked& c, int64_t outer0, int64_t outer1, int64_t tile0, int64_t tile1, int64_t stride0, int bytes) {
  return make_region(c, outer0, c.mul(c.mul(outer1, tile0 * tile1), bytes), outer0 > 0 ? c.mul(stride0, bytes) : 0);
}

uint8_t* written(const Operand& o) { return (uint8_t*)const_cast<void*>(o.dev); }

}  // namespace

UK_API void iree_uk_mi355x_gated_mmt4d_p(const iree_uk_mi355x_gated_mmt4d_params_t* p) {
  tl_last_kernel = "";
  UK_REQUIRE(p != nullptr);
  const bool load = p->flags & IREE_UK_MI355X_FLAG_GATED_MMT4D_PRE_LOAD, store = p->flags & IREE_UK_MI355X_FLAG_GATED_MMT4D_PRE_STORE;
  const bool pre = load || store;
  UK_REQUIRE(gated_flags_known(p->flags, IREE_UK_MI355X_FLAG_GATED_MMT4D_PRE_LOAD | IREE_UK_MI355X_FLAG_GATED_MMT4D_PRE_STORE));
  UK_REQUIRE(pre || !(p->flags & IREE_UK_MI355X_FLAG_GATED_MMT4D_PRE_F32));
  UK_REQUIRE(tile_counts_in_range(p->M, p->N, p->K, p->M0, p->N0, p->K0));
  const uint32_t flag = p->flags & IREE_UK_MI355X_FLAG_GATED_MMT4D_TYPE_MASK;
  const uk::Float type = operand_type_of(flag), out_type = result_type_of(flag),
                  pre_type = p->flags & IREE_UK_MI355X_FLAG_GATED_MMT4D_PRE_F32 ? uk::Float::kF32 : type;
  if (p->M == 0 || p->N == 0 || p->M0 == 0 || p->N0 == 0) return;

  Checked c;
  const int e = uk::float_bytes(out_type), pe = uk::float_bytes(pre_type);
  const RowRegion lhs_region = tiled_region(c, p->M, p->K, p->M0, p->K0, p->lhs_stride0, 2);
  const RowRegion gate_region = tiled_region(c, p->N, p->K, p->N0, p->K0, p->gate_stride0, 2);
  const RowRegion up_region = tiled_region(c, p->N, p->K, p->N0, p->K0, p->up_stride0, 2);
  const RowRegion gate_pre_region = tiled_region(c, pre ? p->M : 0, p->N, p->M0, p->N0, p->gate_pre_stride0, pe);
  const RowRegion up_pre_region = tiled_region(c, pre ? p->M : 0, p->N, p->M0, p->N0, p->up_pre_stride0, pe);
  const RowRegion out_region = tiled_region(c, p->M, p->N, p->M0, p->N0, p->out_stride0, e);
  const int64_t lhs_offset = c.mul(p->lhs_offset, 2), gate_offset = c.mul(p->gate_offset, 2), up_offset = c.mul(p->up_offset, 2),
                gate_pre_offset = c.mul(pre ? p->gate_pre_offset : 0, pe), up_pre_offset = c.mul(pre ? p->up_pre_offset : 0, pe),
                out_offset = c.mul(p->out_offset, e);
  UK_REQUIRE(c.ok && "operand extents fit int64");
  UK_REQUIRE(p->M == 1 || p->lhs_stride0 >= 0);
  UK_REQUIRE(p->N == 1 || (p->gate_stride0 >= 0 && p->up_stride0 >= 0));
  UK_REQUIRE(!pre || p->M == 1 || (p->gate_pre_stride0 >= 0 && p->up_pre_stride0 >= 0));
  UK_REQUIRE(rows_apart(out_region));
  UK_REQUIRE(!store || (rows_apart(gate_pre_region) && rows_apart(up_pre_region)));

  hipStream_t stream = tl_stream;
  Stager stager;
  Operand o_lhs{offset_pointer(p->lhs_buffer, lhs_offset), as_copied(lhs_region), true};
  Operand o_gate{offset_pointer(p->gate_buffer, gate_offset), as_copied(gate_region), true};
  Operand o_up{offset_pointer(p->up_buffer, up_offset), as_copied(up_region), true};
  Operand o_gate_pre{offset_pointer(p->gate_pre_buffer, gate_pre_offset), as_copied(gate_pre_region), load};
  Operand o_up_pre{offset_pointer(p->up_pre_buffer, up_pre_offset), as_copied(up_pre_region), load};
  Operand o_out{offset_pointer(p->out_buffer, out_offset), out_region, false};
  UK_REQUIRE(given(o_lhs, p->lhs_buffer));
  UK_REQUIRE(given(o_gate, p->gate_buffer));
  UK_REQUIRE(given(o_up, p->up_buffer));
  UK_REQUIRE(given(o_gate_pre, p->gate_pre_buffer));
  UK_REQUIRE(given(o_up_pre, p->up_pre_buffer));
  UK_REQUIRE(given(o_out, p->out_buffer));
  Operand* const operands[] = {&o_lhs, &o_gate, &o_up, &o_gate_pre, &o_up_pre, &o_out};
  for (int i = 0; i < 5; ++i) UK_REQUIRE(!overlap(o_out, *operands[i]));
  for (int i = 0; store && i < 3; ++i) UK_REQUIRE(!overlap(o_gate_pre, *operands[i]) && !overlap(o_up_pre, *operands[i]));
  UK_REQUIRE(!store || !overlap(o_gate_pre, o_up_pre));
  if (!stage_operands(stager, operands, 6, stream)) {
    abandon(stager, stream);
    return;
  }
  uk::GatedArgs a;
  a.lhs = (const uint8_t*)o_lhs.dev; a.gate = (const uint8_t*)o_gate.dev; a.up = (const uint8_t*)o_up.dev;
  a.gate_pre = pre ? written(o_gate_pre) : nullptr; a.up_pre = pre ? written(o_up_pre) : nullptr;
  a.out = written(o_out);
  a.lhs_stride0 = p->lhs_stride0; a.gate_stride0 = p->gate_stride0; a.up_stride0 = p->up_stride0;
  a.gate_pre_stride0 = pre ? p->gate_pre_stride0 : 0; a.up_pre_stride0 = pre ? p->up_pre_stride0 : 0;
  a.out_stride0 = p->out_stride0;
  a.M = p->M; a.N = p->N; a.K = p->K0 == 0 ? 0 : p->K;
  a.M0 = p->M0; a.N0 = p->N0; a.K0 = p->K0;
  a.type = type; a.out_type = out_type; a.pre_type = pre_type;
  a.activation = activation_of(p->flags);
  a.pre_load = load; a.pre_store = store;
  if (!launch_ok(uk::launch_gated_mmt4d(a, stream, &tl_last_kernel), "gated_mmt4d")) {
    abandon(stager, stream);
    return;
  }
  const Operand* const outs[] = {&o_out, &o_gate_pre, &o_up_pre};
  finish(stager, stream, outs, store ? 3 : 1);
}

namespace {

// What a backward call's checks and the size of its workspace have in common; null: refused, or (`empty`) nothing to do.
bool gated_backward_args(const iree_uk_mi355x_gated_mmt4d_backward_params_t* p, uk::GatedBackwardArgs* a, bool* empty) {
  *empty = false;
  UK_REQUIRE_TRUE(p != nullptr);
  UK_REQUIRE_TRUE(gated_flags_known(p->flags, IREE_UK_MI355X_FLAG_GATED_MMT4D_ACCUMULATE));
  UK_REQUIRE_TRUE(tile_counts_in_range(p->M, p->N, p->K, p->M0, p->N0, p->K0));
  const uint32_t flag = p->flags & IREE_UK_MI355X_FLAG_GATED_MMT4D_TYPE_MASK;
  const bool of_lhs = p->lhs_grad_buffer, of_gate = p->gate_grad_buffer, of_up = p->up_grad_buffer;
  *a = uk::GatedBackwardArgs();
  a->lhs_grad = (uint8_t*)p->lhs_grad_buffer; a->gate_grad = (uint8_t*)p->gate_grad_buffer; a->up_grad = (uint8_t*)p->up_grad_buffer;
  a->lhs_stride0 = p->lhs_stride0; a->gate_stride0 = p->gate_stride0; a->up_stride0 = p->up_stride0;
  a->gate_pre_stride0 = p->gate_pre_stride0; a->up_pre_stride0 = p->up_pre_stride0; a->out_grad_stride0 = p->out_grad_stride0;
  a->lhs_grad_stride0 = of_lhs ? p->lhs_grad_stride0 : 0;
  a->gate_grad_stride0 = of_gate ? p->gate_grad_stride0 : 0;
  a->up_grad_stride0 = of_up ? p->up_grad_stride0 : 0;
  // (Without rows there are sums over none, without columns too.)
  const bool rows = p->M > 0 && p->M0 > 0, cols = p->N > 0 && p->N0 > 0;
  a->M = rows ? p->M : 0; a->N = cols ? p->N : 0; a->K = p->K;
  a->M0 = p->M0; a->N0 = p->N0; a->K0 = p->K0;
  a->type = operand_type_of(flag); a->out_type = result_type_of(flag);
  a->pre_type = p->flags & IREE_UK_MI355X_FLAG_GATED_MMT4D_PRE_F32 ? uk::Float::kF32 : a->type;
  a->activation = activation_of(p->flags);
  a->accumulate = p->flags & IREE_UK_MI355X_FLAG_GATED_MMT4D_ACCUMULATE;
  *empty = p->K == 0 || p->K0 == 0 || (!rows && !cols) || !(of_lhs || of_gate || of_up) || (!rows && (a->accumulate || !(of_gate || of_up))) ||
           (!cols && !of_lhs);
  return true;
}

}  // namespace

UK_API iree_uk_index_t iree_uk_mi355x_gated_mmt4d_backward_workspace(const iree_uk_mi355x_gated_mmt4d_backward_params_t* p) {
  uk::GatedBackwardArgs a;
  bool empty;
  if (!gated_backward_args(p, &a, &empty) || empty) return 0;
  const int64_t bytes = uk::gated_backward_workspace(a);
  if (bytes < 0) {
    report_failure(__FILE__, __LINE__, __func__, "the workspace fits int64");
    return 0;
  }
  return bytes;
}

UK_API void iree_uk_mi355x_gated_mmt4d_backward_p(const iree_uk_mi355x_gated_mmt4d_backward_params_t* p) {
  tl_last_kernel = "";
  uk::GatedBackwardArgs a;
  bool empty;
  if (!gated_backward_args(p, &a, &empty) || empty) return;
  const bool of_lhs = a.lhs_grad, of_gate = a.gate_grad, of_up = a.up_grad, of_weights = of_gate || of_up;
  const int64_t needed = uk::gated_backward_workspace(a);
  UK_REQUIRE(needed >= 0 && "the workspace fits int64");
  UK_REQUIRE(p->workspace_size >= needed);
  UK_REQUIRE(needed == 0 || p->workspace_buffer != nullptr);
  UK_REQUIRE((uintptr_t)p->workspace_buffer % 256 == 0 || needed == 0);

  Checked c;
  const int e = uk::float_bytes(a.out_type), pe = uk::float_bytes(a.pre_type);
  const int64_t k = p->K, m0 = p->M0, n0 = p->N0, k0 = p->K0;
  const RowRegion lhs_region = tiled_region(c, of_weights ? a.M : 0, k, m0, k0, a.lhs_stride0, 2);
  const RowRegion gate_region = tiled_region(c, of_lhs ? a.N : 0, k, n0, k0, a.gate_stride0, 2);
  const RowRegion up_region = tiled_region(c, of_lhs ? a.N : 0, k, n0, k0, a.up_stride0, 2);
  const RowRegion gate_pre_region = tiled_region(c, a.M, a.N, m0, n0, a.gate_pre_stride0, pe);
  const RowRegion up_pre_region = tiled_region(c, a.M, a.N, m0, n0, a.up_pre_stride0, pe);
  const RowRegion out_grad_region = tiled_region(c, a.M, a.N, m0, n0, a.out_grad_stride0, e);
  const RowRegion lhs_grad_region = tiled_region(c, of_lhs ? a.M : 0, k, m0, k0, a.lhs_grad_stride0, e);
  const RowRegion gate_grad_region = tiled_region(c, of_gate ? a.N : 0, k, n0, k0, a.gate_grad_stride0, e);
  const RowRegion up_grad_region = tiled_region(c, of_up ? a.N : 0, k, n0, k0, a.up_grad_stride0, e);
  const int64_t lhs_offset = c.mul(p->lhs_offset, 2), gate_offset = c.mul(p->gate_offset, 2), up_offset = c.mul(p->up_offset, 2),
                gate_pre_offset = c.mul(p->gate_pre_offset, pe), up_pre_offset = c.mul(p->up_pre_offset, pe),
                out_grad_offset = c.mul(p->out_grad_offset, e), lhs_grad_offset = c.mul(of_lhs ? p->lhs_grad_offset : 0, e),
                gate_grad_offset = c.mul(of_gate ? p->gate_grad_offset : 0, e), up_grad_offset = c.mul(of_up ? p->up_grad_offset : 0, e);
  UK_REQUIRE(c.ok && "operand extents fit int64");
  UK_REQUIRE(a.M <= 1 || (a.lhs_stride0 >= 0 && a.gate_pre_stride0 >= 0 && a.up_pre_stride0 >= 0 && a.out_grad_stride0 >= 0));
  UK_REQUIRE(a.N <= 1 || (a.gate_stride0 >= 0 && a.up_stride0 >= 0));
  UK_REQUIRE(rows_apart(lhs_grad_region));
  UK_REQUIRE(rows_apart(gate_grad_region));
  UK_REQUIRE(rows_apart(up_grad_region));

  hipStream_t stream = tl_stream;
  Stager stager;
  Operand o_lhs{offset_pointer(p->lhs_buffer, lhs_offset), as_copied(lhs_region), true};
  Operand o_gate{offset_pointer(p->gate_buffer, gate_offset), as_copied(gate_region), true};
  Operand o_up{offset_pointer(p->up_buffer, up_offset), as_copied(up_region), true};
  Operand o_gate_pre{offset_pointer(p->gate_pre_buffer, gate_pre_offset), as_copied(gate_pre_region), true};
  Operand o_up_pre{offset_pointer(p->up_pre_buffer, up_pre_offset), as_copied(up_pre_region), true};
  Operand o_out_grad{offset_pointer(p->out_grad_buffer, out_grad_offset), as_copied(out_grad_region), true};
  Operand o_lhs_grad{offset_pointer(p->lhs_grad_buffer, lhs_grad_offset), lhs_grad_region, false};
  Operand o_gate_grad{offset_pointer(p->gate_grad_buffer, gate_grad_offset), gate_grad_region, a.accumulate};
  Operand o_up_grad{offset_pointer(p->up_grad_buffer, up_grad_offset), up_grad_region, a.accumulate};
  Operand o_workspace{p->workspace_buffer, make_region(c, needed > 0 ? 1 : 0, needed, needed), false};
  Operand* const operands[] = {&o_lhs, &o_gate, &o_up, &o_gate_pre, &o_up_pre, &o_out_grad,
                               &o_lhs_grad, &o_gate_grad, &o_up_grad, &o_workspace};
  const void* const buffers[] = {p->lhs_buffer, p->gate_buffer, p->up_buffer, p->gate_pre_buffer, p->up_pre_buffer, p->out_grad_buffer};
  for (int i = 0; i < 6; ++i) UK_REQUIRE(given(*operands[i], buffers[i]));
  for (int i = 6; i < 10; ++i)
    for (int j = 0; j < i; ++j) UK_REQUIRE(!overlap(*operands[i], *operands[j]));
  if (!stage_operands(stager, operands, 10, stream)) {
    abandon(stager, stream);
    return;
  }
  a.lhs = (const uint8_t*)o_lhs.dev; a.gate = (const uint8_t*)o_gate.dev; a.up = (const uint8_t*)o_up.dev;
  a.gate_pre = (const uint8_t*)o_gate_pre.dev; a.up_pre = (const uint8_t*)o_up_pre.dev;
  a.out_grad = (const uint8_t*)o_out_grad.dev;
  a.lhs_grad = of_lhs ? written(o_lhs_grad) : nullptr;
  a.gate_grad = of_gate ? written(o_gate_grad) : nullptr;
  a.up_grad = of_up ? written(o_up_grad) : nullptr;
  a.workspace = written(o_workspace);
  if (!launch_ok(uk::launch_gated_backward(a, stream, &tl_last_kernel), "gated_mmt4d_backward")) {
    abandon(stager, stream);
    return;
  }
  const Operand* const outs[] = {&o_lhs_grad, &o_gate_grad, &o_up_grad};
  finish(stager, stream, outs, 3);
}

namespace {

bool adapter_args(const iree_uk_mi355x_adapter_mmt4d_params_t* p, uk::AdapterArgs* a, bool* empty) {
  *empty = false;
  UK_REQUIRE_TRUE(p != nullptr);
  const uint32_t flag = p->flags & IREE_UK_MI355X_FLAG_ADAPTER_MMT4D_TYPE_MASK;
  UK_REQUIRE_TRUE(!(p->flags & ~(uint32_t)(IREE_UK_MI355X_FLAG_ADAPTER_MMT4D_TYPE_MASK | IREE_UK_MI355X_FLAG_ADAPTER_MMT4D_ACCUMULATE)));
  UK_REQUIRE_TRUE(flag >= IREE_UK_MI355X_FLAG_ADAPTER_MMT4D_TYPE_F16F16F32 && flag <= IREE_UK_MI355X_FLAG_ADAPTER_MMT4D_TYPE_BF16BF16BF16);
  UK_REQUIRE_TRUE(tile_counts_in_range(p->M, p->N, p->K, p->M0, p->N0, p->K0));
  UK_REQUIRE_TRUE(p->M * p->M0 <= 0x7FFFFFFF);
  UK_REQUIRE_TRUE(in_unsigned_range(p->rank, 15));
  UK_REQUIRE_TRUE(in_unsigned_range(p->count, 31));
  *a = uk::AdapterArgs();
  a->lhs_stride0 = p->lhs_stride0; a->out_stride0 = p->out_stride0;
  a->down_stride0 = p->down_stride0; a->down_stride1 = p->down_stride1;
  a->up_stride0 = p->up_stride0; a->up_stride1 = p->up_stride1;
  a->M = p->M; a->N = p->N; a->K = p->K0 == 0 ? 0 : p->K;
  a->M0 = p->M0; a->N0 = p->N0; a->K0 = p->K0;
  a->rank = p->rank; a->count = p->count;
  if (a->K == 0 || a->rank == 0) a->count = 0;  // (nobody has an adapter)
  a->type = operand_type_of(flag); a->out_type = result_type_of(flag);
  a->accumulate = p->flags & IREE_UK_MI355X_FLAG_ADAPTER_MMT4D_ACCUMULATE;
  *empty = p->M == 0 || p->N == 0 || p->M0 == 0 || p->N0 == 0 || (a->accumulate && a->count == 0);
  return true;
}

}  // namespace

UK_API iree_uk_index_t iree_uk_mi355x_adapter_mmt4d_workspace(const iree_uk_mi355x_adapter_mmt4d_params_t* p) {
  uk::AdapterArgs a;
  bool empty;
  if (!adapter_args(p, &a, &empty) || empty) return 0;
  const int64_t bytes = uk::adapter_workspace(a);
  if (bytes < 0) {
    report_failure(__FILE__, __LINE__, __func__, "the workspace fits int64");
    return 0;
  }
  return bytes;
}

UK_API void iree_uk_mi355x_adapter_mmt4d_p(const iree_uk_mi355x_adapter_mmt4d_params_t* p) {
  tl_last_kernel = "";
  uk::AdapterArgs a;
  bool empty;
  if (!adapter_args(p, &a, &empty) || empty) return;
  const int64_t needed = uk::adapter_workspace(a);
  UK_REQUIRE(needed >= 0 && "the workspace fits int64");
  UK_REQUIRE(p->workspace_size >= needed);
  UK_REQUIRE(needed == 0 || p->workspace_buffer != nullptr);
  UK_REQUIRE((uintptr_t)p->workspace_buffer % 256 == 0 || needed == 0);

  Checked c;
  const int e = uk::float_bytes(a.out_type);
  const bool any = a.count > 0;
  const int64_t depth = c.mul(a.K, a.K0), cols = a.N * a.N0, rows = a.M * a.M0;
  UK_REQUIRE(!any || (p->down_stride0 >= 0 && p->down_stride1 >= 0 && p->up_stride0 >= 0 && p->up_stride1 >= 0));
  const RowRegion lhs_region = tiled_region(c, any ? a.M : 0, a.K, a.M0, a.K0, a.lhs_stride0, 2);
  const RowRegion down_region =
      make_region(c, any ? a.count : 0, c.mul(c.add(c.mul(a.rank - 1, any ? a.down_stride1 : 0), depth), 2), c.mul(any ? a.down_stride0 : 0, 2));
  const RowRegion up_region =
      make_region(c, any ? a.count : 0, c.mul(c.add(c.mul(cols - 1, any ? a.up_stride1 : 0), a.rank), 2), c.mul(any ? a.up_stride0 : 0, 2));
  const RowRegion index_region = make_region(c, any ? 1 : 0, rows * 4, 0);
  const RowRegion scales_region = make_region(c, any && p->scales_buffer ? 1 : 0, a.count * 4, 0);
  const RowRegion out_region = tiled_region(c, a.M, a.N, a.M0, a.N0, a.out_stride0, e);
  const int64_t lhs_offset = c.mul(p->lhs_offset, 2), down_offset = c.mul(p->down_offset, 2), up_offset = c.mul(p->up_offset, 2),
                index_offset = c.mul(p->index_offset, 4), scales_offset = c.mul(p->scales_buffer ? p->scales_offset : 0, 4),
                out_offset = c.mul(p->out_offset, e);
  UK_REQUIRE(c.ok && "operand extents fit int64");
  UK_REQUIRE(a.M == 1 || a.lhs_stride0 >= 0);
  UK_REQUIRE(rows_apart(out_region));

  hipStream_t stream = tl_stream;
  Stager stager;
  Operand o_lhs{offset_pointer(p->lhs_buffer, lhs_offset), as_copied(lhs_region), true};
  Operand o_down{offset_pointer(p->down_buffer, down_offset), as_copied(down_region), true};
  Operand o_up{offset_pointer(p->up_buffer, up_offset), as_copied(up_region), true};
  Operand o_index{offset_pointer(p->index_buffer, index_offset), index_region, true};
  Operand o_scales{offset_pointer(p->scales_buffer, scales_offset), scales_region, true};
  Operand o_out{offset_pointer(p->out_buffer, out_offset), out_region, a.accumulate};
  Operand o_workspace{p->workspace_buffer, make_region(c, needed > 0 ? 1 : 0, needed, needed), false};
  Operand* const operands[] = {&o_lhs, &o_down, &o_up, &o_index, &o_scales, &o_out, &o_workspace};
  const void* const buffers[] = {p->lhs_buffer, p->down_buffer, p->up_buffer, p->index_buffer, p->scales_buffer, p->out_buffer};
  for (int i = 0; i < 6; ++i) UK_REQUIRE(given(*operands[i], buffers[i]));
  UK_REQUIRE((uintptr_t)o_index.ptr % 4 == 0 && (uintptr_t)o_scales.ptr % 4 == 0);
  for (int i = 5; i < 7; ++i)
    for (int j = 0; j < i; ++j) UK_REQUIRE(!overlap(*operands[i], *operands[j]));
  if (!stage_operands(stager, operands, 7, stream)) {
    abandon(stager, stream);
    return;
  }
  a.lhs = (const uint8_t*)o_lhs.dev; a.down = (const uint8_t*)o_down.dev; a.up = (const uint8_t*)o_up.dev;
  a.index = (const int32_t*)o_index.dev;
  a.scales = any && p->scales_buffer ? (const float*)o_scales.dev : nullptr;
  a.out = written(o_out);
  a.workspace = written(o_workspace);
  if (!launch_ok(uk::launch_adapter_mmt4d(a, stream, &tl_last_kernel), "adapter_mmt4d")) {
    abandon(stager, stream);
    return;
  }
  finish(stager, stream, o_out);
}

//===----------------------------------------------------------------------===//
// Entry points without a reference counterpart
//===----------------------------------------------------------------------===//

UK_API int iree_uk_mi355x_multi_mma_i32_16x16x64_i8(const void* a, const void* b, void* c, long long outer_m,
                                                    long long outer_n, int32_t k_size, int32_t intrinsics_m,
                                                    int32_t subgroups_m, int32_t intrinsics_n, int32_t subgroups_n,
                                                    int32_t intrinsics_k) {
  tl_last_kernel = "";
  // Device pointers only: the data-tiled operands of a GPU dispatch never live on the host.
  if (!device_accessible(a) || !device_accessible(b) || !device_accessible(c)) return (int)hipErrorInvalidValue;
  const hipError_t e = uk::launch_multi_mma_i8(a, b, c, outer_m, outer_n, k_size, intrinsics_m, subgroups_m,
                                               intrinsics_n, subgroups_n, intrinsics_k, tl_stream);
  if (e != hipSuccess) return (int)e;
  tl_last_kernel = "multi_mma_i32_16x16x64_i8";
  if (!tl_async) {
    const hipError_t s = hipStreamSynchronize(tl_stream);
    if (s != hipSuccess) return (int)s;
  }
  return 0;
}

UK_API int iree_uk_mi355x_version(void) { return 100; }

UK_API int iree_uk_mi355x_init(int device_ordinal) {
  hipError_t e = device_ordinal < 0 ? hipGetDevice(&device_ordinal) : hipSetDevice(device_ordinal);
  if (e != hipSuccess) return (int)e;
  hipDeviceProp_t prop;
  e = hipGetDeviceProperties(&prop, device_ordinal);
  if (e != hipSuccess) return (int)e;
  if (strncmp(prop.gcnArchName, "gfx950", 6) != 0) return (int)hipErrorInvalidDevice;
  // Resolve this device's static staging memory now, so that the
  // allocation-free entry point does nothing but copies and launches.
  if (device_ordinal < kMaxDevices && hipSetDevice(device_ordinal) == hipSuccess &&
      !scratch_for_current_device())
    return (int)hipErrorInvalidSymbol;
  return 0;
}

UK_API void iree_uk_mi355x_set_stream(void* stream, int asynchronous) {
  tl_stream = (hipStream_t)stream;
  tl_async = asynchronous != 0;
}

UK_API void iree_uk_mi355x_set_fail_handler(iree_uk_mi355x_fail_handler_t handler) {
  g_fail_handler.store(handler, std::memory_order_release);
}

UK_API const char* iree_uk_mi355x_last_kernel(void) { return tl_last_kernel; }
