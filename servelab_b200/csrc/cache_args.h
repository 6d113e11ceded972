// Arguments of the kernels over caches in the compute type or in 8 bits, as the host checks and fills them in.
#pragma once

enum { CACHE_PLAIN = 0, CACHE_INT8 = 1, CACHE_E4M3 = 2 };

struct CacheWriteArgs {
    const void* qkv; long long ld;
    const float* bias;
    const int* pos; const int* slots;            // slots may be null: the positions
    const int* seq; const int* table;
    int max_pages, num_seqs, ps, num_pages;
    const float* inv_freq; int rot;
    void* q_out; long long ldq;
    void* k; void* v; float* ks; float* vs;
    int T, H, Hkv, D, kind;
    int exact;                                   // angles in 64 bits; 0: rounded to float32, as the other writers' are
};
struct CacheReadArgs {
    const void* k; const void* v; const float* ks; const float* vs;
    const int* table; int max_pages, num_seqs, ps, num_pages;
    const int* first; const int* cu;
    void* k_out; void* v_out; long long ldk, ldv;        // elements between the rows of two tokens
    int rows, Hkv, D, kind;
};
struct CacheAttnArgs {
    const void* q; long long ldq;
    void* out; long long ldo;
    const void* k; const void* v; const float* ks; const float* vs;
    const int* table; int max_pages;
    const int* cu_q; const int* ctx_len;
    const int* mask; int mask_words;             // null: causal
    const int* pos;                              // with a mask and a window; otherwise may be null
    float* part_o; float* part_ml;               // [T H][parts][D], [T H][parts][2], with parts > 1
    int parts;                                   // partial results a row; 1: none, `out` is written
    int T, S, H, Hkv, D, ps, num_pages, kind, window;
    float scale;
    int tiles;                                   // tiles of rows a request has at most, as far as the caller knows
    int cluster;                                 // blocks of a cluster that share a tile's keys
    int more;                                    // units of the kernel for many rows with one part more
};
