// Which kernel shrinks the rows, beside whether the product takes them in the order of their adapters:
// what it reads there must have been written.  Every number of rows that the few rows' kernel may take and
// some past it, every width of the shrunk values (slices x rank) with its number of slices, few and many slots.
#include "launches.h"

#include "../../nano-vllm-extend_amd/csrc/lora.hip"

extern "C" int gdn_quantize_fp8(const void*, int, int64_t, uint8_t*, int64_t, float*, int64_t, int64_t, int64_t, int, int, void*) {
  return GDN_OK;
}

int main() {
  const void* wrote = nullptr;  // the kernel, where it writes the order
  int shrinks = 0, bad = 0, calls = 0, sorted = 0;
  dim3 grid;
  launches::seen = [&](const void* f, const dim3& g, const dim3&, void**) {
    ++shrinks;
    grid = g;
    const bool orders = f == reinterpret_cast<const void*>(&lora_few_kernel<false, true>) ||
                        f == reinterpret_cast<const void*>(&lora_few_kernel<true, true>);
    wrote = orders ? f : nullptr;
  };
  auto* const p = reinterpret_cast<uint16_t*>(uintptr_t{1} << 20);
  auto* const f = reinterpret_cast<float*>(p);
  auto* const i = reinterpret_cast<int32_t*>(p);
  auto* const b = reinterpret_cast<uint8_t*>(p);
  const int K = 128;
  for (int M = 1; M <= 2112; ++M)
    for (int slices = 1; slices <= kMaxParts; ++slices)
      for (int rank = 8; rank <= kMaxRank; rank += 8)
        for (int slots : {1, 64, (1 << 23) - 1, 1 << 23})
          for (int form = 0; form < 3; ++form) {  // bf16 rows, bf16 rows quantized on the way, e4m3 rows
            const int cols = slices * rank, x_bf16 = form < 2;
            wrote = nullptr;
            shrinks = 0;
            const int status = gdn_lora_shrink(p, x_bf16, K, f, 1, M, p, int64_t{cols} * K, f, i, slots, slices, rank, M, K, p,
                                               2 * cols, i, form == 1 ? b : nullptr, K, f, 1, M, nullptr);
            // the widths of the slices are the product's own affair
            const int ends[4] = {16, 32, 48, 64};
            Lora lo{};
            const bool ok = lora_of(lo, p, 2 * cols, i, p, 64LL * rank, i, slots, rank, slices, ends, M, 16 * slices);
            // (the order follows the groups)
            const bool reads = lo.order != nullptr;
            ++calls;
            sorted += reads;
            if (status != GDN_OK || !ok || shrinks != 1 || reads != (wrote != nullptr) || grid.x < 1 || grid.y < 1 ||
                grid.y > 65535 || (reads && lo.order != i + (M + 15) / 16)) {
              if (bad++ < 5)
                std::printf("M %d slices %d rank %d slots %d form %d: status %d, product's arguments %d, launches %d, order read "
                            "%d, written %d\n", M, slices, rank, slots, form, status, ok, shrinks, reads, wrote != nullptr);
            }
          }
  std::printf("%d of %d calls, %d in order\n", bad, calls, sorted);
  return bad != 0 || sorted == 0;
}
