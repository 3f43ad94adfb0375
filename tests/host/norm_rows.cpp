// The launches of the norm around a block: each of fewer than 2^32 threads, together every row once, with each operand's
// rows where they are.  Rows of every launch's width, up to the most that the entry point takes.
#include "launches.h"

#include "../../nano-vllm-extend_amd/csrc/block_norm.hip"

int main() {
  int bad = 0, calls = 0, several = 0;
  const uintptr_t base = uintptr_t{1} << 20;
  auto* const p = reinterpret_cast<uint16_t*>(base);
  for (int H : {1, 8, 128, 1000, 1024, 1025, 2048, 2176, 4096, 4224, 16384})
    for (int64_t M : {int64_t{1}, int64_t{5}, int64_t{2048}, int64_t{4194303}, int64_t{4194305}, int64_t{1} << 23, (int64_t{1} << 24) - 1,
                      int64_t{1} << 24, (int64_t{1} << 24) + 1, (int64_t{1} << 26) - 4, int64_t{1} << 26, (int64_t{1} << 26) + 5,
                      (int64_t{1} << 31) - 1})
      for (int form = 0; form < 16; ++form) {
        const bool f32 = form & 1, e4m3 = (form & 2) && H % 128 == 0, full = form & 4, bare = form & 8;
        const int64_t wide = full ? H + 8 : H;  // the rows' stride
        int64_t rows = 0;
        int launched = 0;
        bool ok = true;
        launches::seen = [&](const void*, const dim3& grid, const dim3& block, void** args) {
          const NormArgs& a = *static_cast<const NormArgs*>(args[0]);
          ++launched;
          ok = ok && static_cast<uint64_t>(grid.x) * block.x < (uint64_t{1} << 32) && grid.y == 1 && grid.z == 1 && a.M > 0;
          const int64_t waves = static_cast<int64_t>(block.x) / 64;
          // (a wave to a row, or a workgroup to one)
          ok = ok && (a.M + waves - 1) / waves <= grid.x && grid.x <= a.M;
          auto at = [&](const void* q, int64_t bytes) { return reinterpret_cast<uintptr_t>(q) == base + static_cast<uint64_t>(rows * bytes); };
          ok = ok && at(a.x, 2 * wide) && a.H == H && a.sx == wide;
          ok = ok && (bare ? !a.residual : at(a.residual, (f32 ? 4 : 2) * wide)) && at(a.stream, (f32 && !bare ? 4 : 2) * H);
          ok = ok && at(a.y, 2 * H) && (e4m3 ? at(a.y8, H) && at(a.y8_scale, 4) : !a.y8 && !a.y8_scale);
          ok = ok && at(a.gate, (f32 ? 4 : 2) * (full ? H : 1)) && at(a.w, 0) && at(a.post_w, 0);
          rows += a.M;
        };
        const int status = gdn_add_rms_norm(p, wide, bare ? nullptr : p, wide, f32 && !bare, p, p, f32, 1.0f, p, f32, full ? H : 1, full,
                                            0, 1.0f, 1e-6f, p, p, e4m3 ? reinterpret_cast<uint8_t*>(p) : nullptr,
                                            e4m3 ? reinterpret_cast<float*>(p) : nullptr, 1, M, M, H, nullptr);
        ++calls;
        several += launched > 1;
        if (status != GDN_OK || !ok || rows != M || !launched) {
          if (bad++ < 5)
            std::printf("M %lld H %d form %d: status %d, %d launches of %lld rows, as they should be %d\n", static_cast<long long>(M), H,
                        form, status, launched, static_cast<long long>(rows), ok);
        }
      }
  std::printf("%d of %d calls, %d in several launches\n", bad, calls, several);
  return bad != 0 || several == 0;
}
