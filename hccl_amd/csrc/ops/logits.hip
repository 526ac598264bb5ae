// Checks and tables of logits whose columns are split over the ranks (ops/logits.h).
#include "ops/logits.h"

namespace hcclx {
namespace logits {

namespace {

uint64_t address(const void *p) { return reinterpret_cast<uint64_t>(p); }

int check_pointers(const hcclx_logits_t &l, const void *const *p, const char *what)
{
    if (p == nullptr) return fail(HCCL_E_PTR, std::string(what) + " pointer array is null");
    const uint64_t size = dtype_size(l.dtype);
    for (uint32_t j = 0; j < l.n; ++j) {
        if (l.columns[j] == 0) continue;
        if (p[j] == nullptr) return fail(HCCL_E_PTR, std::string(what) + "[" + std::to_string(j) + "] is null");
        if (address(p[j]) % size != 0) {
            return fail(HCCL_E_PARA, std::string(what) + "[" + std::to_string(j) + "] is not aligned to " + std::to_string(size) + " bytes");
        }
    }
    return HCCL_SUCCESS;
}

// Whether rows of `a` bytes every `step` bytes from p and rows of `b` bytes every `other_step` bytes from q have no byte in common.
// (Ranks' columns of one matrix lie side by side: their rows interleave.)
bool apart(uint64_t p, uint64_t a, uint64_t step, uint64_t a_extent, uint64_t q, uint64_t b, uint64_t other_step, uint64_t b_extent)
{
    if (p >= q + b_extent || q >= p + a_extent) return true;
    if (step != other_step || a > step || b > step) return false;
    const uint64_t behind = p >= q ? (p - q) % step : (step - (q - p) % step) % step;
    return behind >= b && behind + a <= step;
}

}  // namespace

uint64_t stride(const hcclx_logits_t &l, uint32_t j)
{
    return (l.row_stride == nullptr ? l.columns[j] : l.row_stride[j]) * dtype_size(l.dtype);
}

uint64_t extent(const hcclx_logits_t &l, uint32_t j)
{
    if (l.rows == 0 || l.columns[j] == 0) return 0;
    return (l.rows - 1) * stride(l, j) + static_cast<uint64_t>(l.columns[j]) * dtype_size(l.dtype);
}

int check(const hcclx_logits_t &l, void *const *to, uint32_t *vocab)
{
    if (l.n == 0 || l.n > kMostRanks) return fail(HCCL_E_PARA, "rank count outside 1.." + std::to_string(kMostRanks));
    if (l.dtype != HCCL_DATA_TYPE_FP32 && l.dtype != HCCL_DATA_TYPE_FP16 && l.dtype != HCCL_DATA_TYPE_BFP16) {
        return fail(HCCL_E_NOT_SUPPORT, "logits are fp32, fp16 or bf16");
    }
    if (l.rows > kMostRows) return fail(HCCL_E_PARA, "more rows than " + std::to_string(kMostRows));
    if (l.columns == nullptr) return fail(HCCL_E_PTR, "columns is null");
    uint64_t sum = 0;
    for (uint32_t j = 0; j < l.n; ++j) {
        sum += l.columns[j];
        if (l.row_stride == nullptr) continue;
        if (l.row_stride[j] < l.columns[j] && l.rows > 1) return fail(HCCL_E_PARA, "rows of rank " + std::to_string(j) + " overlap");
        if (l.row_stride[j] >> 32 != 0) return fail(HCCL_E_PARA, "row stride of rank " + std::to_string(j) + " is 2^32 or more");
    }
    if (sum == 0 || sum > HCCLX_LOGITS_MAX_COLUMNS) {
        return fail(HCCL_E_PARA, "columns of all ranks together outside 1.." + std::to_string(HCCLX_LOGITS_MAX_COLUMNS));
    }
    int rc = check_pointers(l, l.logits, "logits");
    if (rc == HCCL_SUCCESS && to != nullptr) rc = check_pointers(l, to, "dlogits");
    *vocab = static_cast<uint32_t>(sum);
    return rc;
}

int check_array(const void *p, uint64_t align, bool optional, const char *what)
{
    if (p == nullptr) return optional ? HCCL_SUCCESS : fail(HCCL_E_PTR, std::string(what) + " is null");
    if (address(p) % align != 0) return fail(HCCL_E_PARA, std::string(what) + " is not aligned to " + std::to_string(align) + " bytes");
    return HCCL_SUCCESS;
}

int check_apart(const char *what, const void *p, uint64_t bytes, const char *other, const void *q, uint64_t other_bytes)
{
    if (p == nullptr || q == nullptr || bytes == 0 || other_bytes == 0) return HCCL_SUCCESS;
    if (address(p) >= address(q) + other_bytes || address(q) >= address(p) + bytes) return HCCL_SUCCESS;
    return fail(HCCL_E_PARA, std::string(what) + " overlaps " + other);
}

int check_apart(const hcclx_logits_t &l, const char *of_what, const void *const *of, const char *what, const void *p, uint64_t bytes)
{
    if (p == nullptr || of == nullptr || bytes == 0) return HCCL_SUCCESS;
    for (uint32_t j = 0; j < l.n; ++j) {
        const uint64_t held = extent(l, j);
        if (held == 0) continue;
        // (a single stretch: rows of its own length, a whole distance apart)
        if (apart(address(p), bytes, stride(l, j), bytes, address(of[j]), l.columns[j] * dtype_size(l.dtype), stride(l, j), held)) continue;
        return fail(HCCL_E_PARA, std::string(what) + " overlaps " + of_what + "[" + std::to_string(j) + "]");
    }
    return HCCL_SUCCESS;
}

int check_gradients(const hcclx_logits_t &l, void *const *to)
{
    const uint64_t size = dtype_size(l.dtype);
    for (uint32_t i = 0; i < l.n; ++i) {
        for (uint32_t j = 0; j < l.n; ++j) {
            if (extent(l, i) == 0 || extent(l, j) == 0) continue;
            const auto free_of = [&](const void *q) {
                return apart(address(to[i]), l.columns[i] * size, stride(l, i), extent(l, i), address(q), l.columns[j] * size, stride(l, j), extent(l, j));
            };
            if (!(i == j && to[i] == l.logits[j]) && !free_of(l.logits[j])) {
                return fail(HCCL_E_PARA, "dlogits[" + std::to_string(i) + "] overlaps logits[" + std::to_string(j) + "], which others read");
            }
            if (i < j && !free_of(to[j])) {
                return fail(HCCL_E_PARA, "dlogits[" + std::to_string(i) + "] overlaps dlogits[" + std::to_string(j) + "]");
            }
        }
    }
    return HCCL_SUCCESS;
}

int lay_out(const hcclx_logits_t &l, void *const *to, uint32_t vocab, Table *table)
{
    const uint32_t size = dtype_size(l.dtype);
    const uint32_t chunk = 64 * (16 / size);
    std::vector<Stretch> all, ranks;
    uint32_t first = 0;
    for (uint32_t j = 0; j < l.n; ++j) {
        if (l.columns[j] == 0) continue;
        const char *at = static_cast<const char *>(l.logits[j]);
        char *dst = to == nullptr ? nullptr : static_cast<char *>(to[j]);
        const uint64_t step = stride(l, j);
        ranks.push_back({at, dst, step, first, l.columns[j]});
        for (uint32_t c = 0; c < l.columns[j]; c += chunk) {
            const uint64_t o = static_cast<uint64_t>(c) * size;
            all.push_back({at + o, dst == nullptr ? nullptr : dst + o, step, first + c, std::min(chunk, l.columns[j] - c)});
        }
        first += l.columns[j];
    }
    const uint32_t nchunks = static_cast<uint32_t>(all.size());
    all.insert(all.end(), ranks.begin(), ranks.end());
    table->bytes = all.size() * sizeof(Stretch);
    int rc = table->block.get(table->bytes);
    if (rc != HCCL_SUCCESS) return rc;
    HCCLX_HIP(hipMemcpy(table->block.p, all.data(), table->bytes, hipMemcpyHostToDevice));
    const Stretch *held = reinterpret_cast<const Stretch *>(table->block.p);
    table->rows = {held, held + nchunks, nchunks, static_cast<uint32_t>(ranks.size()), l.rows, vocab};
    return HCCL_SUCCESS;
}

}  // namespace logits
}  // namespace hcclx
