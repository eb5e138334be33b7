// Attention by formula and rules: argument checks, tensor maps, choice of the kernel (scored_attn.cuh).
#include "scored_attn.cuh"

namespace stof {
template <>
int launch_scored<64>(const ScoredMaps&, const ScoredParams&, int, bool, int, long long, size_t, cudaStream_t);
template <>
int launch_scored<128>(const ScoredMaps&, const ScoredParams&, int, bool, int, long long, size_t, cudaStream_t);

namespace {

// A 4-D map of (batch, heads, rows, dim) with boxes of box_rows x 64 columns; the outer dimensions in the order of their strides
int make_map(CUtensorMap* map, const void* base, int batch, int heads, int rows, int dim, int box_rows, const long long st[3], int* slot_s, int* slot_h, int* slot_b) {
    struct Dim { uint64_t size; long long stride; int logical; } d[3] = {
        {static_cast<uint64_t>(rows), st[2], 0}, {static_cast<uint64_t>(heads), st[1], 1}, {static_cast<uint64_t>(batch), st[0], 2}};
    for (int i = 0; i < 3; ++i)
        for (int j = i + 1; j < 3; ++j)
            if (d[j].stride < d[i].stride) { Dim t = d[i]; d[i] = d[j]; d[j] = t; }
    uint64_t dims[4] = {static_cast<uint64_t>(dim), 0, 0, 0}, strides[3];
    uint32_t box[4] = {64, 1, 1, 1};
    for (int i = 0; i < 3; ++i) {
        dims[i + 1] = d[i].size;
        strides[i] = static_cast<uint64_t>(d[i].stride) * 2;
        if (d[i].logical == 0) { box[i + 1] = static_cast<uint32_t>(box_rows); *slot_s = i + 1; }
        if (d[i].logical == 1) *slot_h = i + 1;
        if (d[i].logical == 2) *slot_b = i + 1;
    }
    return make_tensor_map_f16(map, base, 4, dims, strides, box);        // (bf16 moves as fp16 does: 16 bits)
}

}  // namespace
}  // namespace stof

using namespace stof;

extern "C" int stof_scored_attn(const void* q, const void* k, const void* v, void* out, int dtype, int batch, int heads, int kv_heads, int q_len, int k_len,
                                int head_dim, const long long q_strides[3], const long long k_strides[3], const long long v_strides[3],
                                const long long out_strides[3], const stof_score_rules* rules, int* status_dev, void* stream_) {
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    STOF_REQUIRE(batch >= 0 && heads > 0 && kv_heads > 0 && q_len >= 0 && k_len >= 0, "scored_attn: bad shape");
    STOF_REQUIRE(heads % kv_heads == 0, "scored_attn: %d heads are not a multiple of %d K/V heads", heads, kv_heads);
    STOF_REQUIRE(head_dim == 64 || head_dim == 128, "scored_attn: head_dim %d not in {64, 128}", head_dim);
    STOF_REQUIRE(dtype == STOF_DTYPE_F16 || dtype == STOF_DTYPE_BF16, "scored_attn: fp16 or bf16 expected");
    STOF_REQUIRE(static_cast<long long>(q_len) + k_len < (1ll << 29), "scored_attn: %d queries and %d keys are beyond 2^29", q_len, k_len);
    STOF_REQUIRE(rules != nullptr, "scored_attn: null rules");
    STOF_REQUIRE(rules->softmax_scale > 0.f && rules->softmax_scale < INFINITY, "scored_attn: softmax_scale must be positive and finite");
    STOF_REQUIRE(rules->softcap >= 0.f && rules->softcap < INFINITY, "scored_attn: softcap must not be negative");
    STOF_REQUIRE(rules->window >= 0, "scored_attn: window must not be negative");
    STOF_REQUIRE(rules->distance_bias == nullptr || (rules->bias_radius >= 0 && rules->bias_radius <= STOF_SCORED_MAX_RADIUS), "scored_attn: bias radius %d beyond %d",
                 rules->bias_radius, STOF_SCORED_MAX_RADIUS);
    STOF_REQUIRE(rules->prefix_lens == nullptr || rules->causal, "scored_attn: a prefix makes keys visible that a causal mask hides: it needs causal");
    if (rules->documents != nullptr) {
        STOF_REQUIRE(q_len <= k_len, "scored_attn: documents name keys: %d queries need as many keys, got %d", q_len, k_len);
        STOF_REQUIRE(rules->documents_stride >= k_len || batch <= 1, "scored_attn: row stride of documents below the number of keys");
        if (k_len > STOF_SCORED_MAX_DOC_KEYS) {
            set_error("scored_attn: documents over %d keys, beyond the maximum of %d", k_len, STOF_SCORED_MAX_DOC_KEYS);
            return STOF_E_LIMIT;
        }
    }
    if (batch == 0 || q_len == 0) return STOF_OK;
    STOF_REQUIRE(k_len > 0, "scored_attn: no keys");
    STOF_REQUIRE(q && k && v && out && q_strides && k_strides && v_strides && out_strides, "scored_attn: null pointer");
    STOF_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(out), "scored_attn: pointers must be 16-byte aligned");
    for (const long long* st : {q_strides, k_strides, v_strides, out_strides})
        for (int i = 0; i < 3; ++i) STOF_REQUIRE(st[i] > 0 && st[i] % 8 == 0, "scored_attn: strides must be positive multiples of 8 elements");
    ScoredParams p;
    p.slopes = rules->slopes; p.distance_bias = rules->distance_bias; p.documents = rules->documents; p.prefix_lens = rules->prefix_lens;
    p.key_lens = rules->key_lens; p.documents_stride = rules->documents_stride; p.status = status_dev;
    p.scale = rules->softmax_scale; p.softcap = usable_cap(rules->softcap); p.causal = rules->causal != 0; p.radius = rules->bias_radius;
    p.window = rules->window > q_len + k_len ? q_len + k_len : rules->window;
    p.batch = batch; p.heads = heads; p.group = heads / kv_heads; p.q_len = q_len; p.k_len = k_len;
    p.table_bytes = rules->distance_bias != nullptr ? (2 * p.radius + 1 + 2 * SA_PAD) * 4 + 4 : 0;       // (an even number of words: pairs follow)
    p.range_bytes = rules->documents != nullptr ? (k_len + SA_T - 1) / SA_T * 8 : 0;
    ScoredMaps maps;
    if (int rc = make_map(&maps[0], q, batch, heads, q_len, head_dim, SA_T, q_strides, &p.slot_s[0], &p.slot_h[0], &p.slot_b[0])) return rc;
    if (int rc = make_map(&maps[1], k, batch, kv_heads, k_len, head_dim, SA_T, k_strides, &p.slot_s[1], &p.slot_h[1], &p.slot_b[1])) return rc;
    if (int rc = make_map(&maps[2], v, batch, kv_heads, k_len, head_dim, SA_T, v_strides, &p.slot_s[2], &p.slot_h[2], &p.slot_b[2])) return rc;
    if (int rc = make_map(&maps[3], out, batch, heads, q_len, head_dim, 32, out_strides, &p.slot_s[3], &p.slot_h[3], &p.slot_b[3])) return rc;
    const long long pairs = static_cast<long long>(batch) * heads;
    // Heads of 64: one half, two blocks on an SM, which cover each other's beginnings and ends (8192 x 32 x 8192: causal 375 us against
    // 388 with two halves, 8 x 1001 with a table 79 against 83).  Heads of 128: two halves share their tiles (859 us against 949), in
    // whole rounds of blocks, though; single halves go round in blocks half as long, of which the last run alone on their SM (2 x 32 x
    // 2048 queries, 3.46 rounds: 128 us against 139).  Costs in rounds of two halves:
    const long long sms = sm_count(), single = pairs * ((q_len + SA_T - 1) / SA_T), doubled = pairs * ((q_len + 2 * SA_T - 1) / (2 * SA_T));
    const long long over = single % (2 * sms);
    const double rounds1 = static_cast<double>(single / (2 * sms)) + (over == 0 ? 0.0 : over <= sms ? 0.62 : 1.0);
    const int halves = head_dim == 64 || 1.07 * rounds1 < static_cast<double>((doubled + sms - 1) / sms) ? 1 : 2;
    p.q_tiles = (q_len + halves * SA_T - 1) / (halves * SA_T);
    STOF_REQUIRE(pairs * p.q_tiles < (1ll << 31), "scored_attn: batch * heads * query tiles beyond 2^31");
    const size_t smem = 1024 + static_cast<size_t>(halves + 2 * scored_slots(head_dim, halves)) * SA_T * head_dim * 2 + p.table_bytes + p.range_bytes;
    int mode = p.slopes != nullptr || p.distance_bias != nullptr ? SA_ANY : p.softcap > 0.f ? SA_CAP : SA_PLAIN;
    if (p.documents != nullptr) mode = (mode == SA_PLAIN ? SA_PLAIN : SA_ANY) | SA_DOCS;
    const bool bf16 = dtype == STOF_DTYPE_BF16;
    return head_dim == 64 ? launch_scored<64>(maps, p, halves, bf16, mode, pairs * p.q_tiles, smem, stream)
                          : launch_scored<128>(maps, p, halves, bf16, mode, pairs * p.q_tiles, smem, stream);
}
