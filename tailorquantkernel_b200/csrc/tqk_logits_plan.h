// tqk_logits_plan.h -- how many CTAs share a row of tqk_process_logits (host only).
#pragma once

namespace tqk {

constexpr int LG_CLUSTER = 16;           // most CTAs per row (non-portable above 8), a power of two
constexpr int LG_CLUSTER_PORTABLE = 8;
constexpr int LG_OWN = 16384;            // tokens per CTA, from which more CTAs take a row

// log2 of the CTAs per row: as few (up to 8) as hold 16384 tokens each, since every one of them scans the row's history,
// and more, up to `most`, while two of all CTAs per SM suffice and each keeps 2048 tokens.  Everything on, histories of up
// to 2000:
//   30001 tokens, 1, 2, 4 and 8 CTAs per row: 10 rows 20.3, 14.6, 11.3, 10.5 us, 74 rows 24.0, 17.0, 18.4, 21.5 us,
//   148 rows 27.3, 22.1, 24.9, 35.8 us, 512 rows 73, 53, 65, 109 us;
//   128256 tokens, 8 and 16 (histories of up to 4000): 1 row 13.7, 10.9 us, 24 rows 15.8, 15.6 us, 37 rows 21.0, 24.9 us
inline int logits_cluster_log(int n_rows, int vocab, int sms, int most) {
    int log_c = 0;
    while (2 << log_c <= most && vocab > 4096 << log_c &&
           ((1 << log_c < LG_CLUSTER_PORTABLE && vocab > LG_OWN << log_c) || (long long)n_rows << (log_c + 1) <= 2LL * sms))
        log_c++;
    return log_c;
}

}  // namespace tqk
