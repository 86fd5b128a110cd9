// What csrc/attention_batch_walk.h and csrc/wave.h need of the HIP runtime, for a test that compiles them with the host
// compiler: a wave is 64 contexts of one thread, run in turn, which meet at every move between lanes.
#pragma once

#include <setjmp.h>
#include <ucontext.h>

#include <algorithm>
#include <cstddef>
#include <cstdint>
#include <cstdlib>
#include <functional>
#include <stdexcept>
#include <string>
#include <vector>

#define __device__
#define __host__
#define __global__
#define __forceinline__ inline

typedef struct ihipStream_t* hipStream_t;

struct float2 {
    float x, y;
};

template <typename T>
inline T min(T a, T b) { return b < a ? b : a; }
template <typename T>
inline T max(T a, T b) { return a < b ? b : a; }

namespace host_wave {

constexpr int kLanes = 64;
constexpr size_t kStack = 128 * 1024;

struct Wave {
    ucontext_t first[kLanes];
    jmp_buf at[kLanes];
    bool begun[kLanes];
    jmp_buf home_at;
    uint32_t value[2][kLanes];
    uint32_t op[2][kLanes];
    uint32_t count[kLanes];   // moves that a lane has made
    int lane;
    const std::function<void(uint32_t)>* body;
    bool bad;
    std::string error;   // what a lane has thrown
    std::vector<char> stacks;
};

inline Wave& wave() {
    static Wave w;
    return w;
}

inline void to_lane(int lane) {
    Wave& w = wave();
    w.lane = lane;
    if (!w.begun[lane]) {
        w.begun[lane] = true;
        setcontext(&w.first[lane]);
    }
    _longjmp(w.at[lane], 1);
}

// This lane's turn ends; the next lane's begins, after the last the first's.
inline void turn() {
    Wave& w = wave();
    if (_setjmp(w.at[w.lane]) == 0) to_lane((w.lane + 1) % kLanes);
}

// The values that all lanes bring to a move. Lanes that meet in different ones have diverged.
inline const uint32_t* meet(uint32_t v, uint32_t op) {
    Wave& w = wave();
    const uint32_t side = w.count[w.lane] & 1u;
    w.value[side][w.lane] = v;
    w.op[side][w.lane] = op;
    ++w.count[w.lane];
    turn();
    for (int i = 0; i < kLanes; ++i)
        if (w.op[side][i] != op) w.bad = true;
    return w.value[side];
}

inline void lane_main() {
    Wave& w = wave();
    const int lane = w.lane;
    try {
        (*w.body)(static_cast<uint32_t>(lane));
    } catch (const std::exception& e) {
        w.error = e.what();
    }
    // All lanes make the same moves, so they end in turn.
    if (w.error.empty() && lane + 1 < kLanes) to_lane(lane + 1);
    _longjmp(w.home_at, 1);
}

// body(lane) for 64 lanes that move values between each other.
inline void run(const std::function<void(uint32_t)>& body) {
    Wave& w = wave();
    if (w.stacks.empty()) w.stacks.resize(kLanes * kStack);
    w.body = &body;
    w.bad = false;
    w.error.clear();
    for (int i = 0; i < kLanes; ++i) {
        w.begun[i] = false;
        w.count[i] = 0u;
        getcontext(&w.first[i]);
        w.first[i].uc_stack.ss_sp = w.stacks.data() + i * kStack;
        w.first[i].uc_stack.ss_size = kStack;
        w.first[i].uc_link = nullptr;
        makecontext(&w.first[i], reinterpret_cast<void (*)()>(lane_main), 0);
    }
    if (_setjmp(w.home_at) == 0) to_lane(0);
    if (!w.error.empty()) throw std::runtime_error(w.error);
    for (int i = 1; i < kLanes; ++i)
        if (w.count[i] != w.count[0]) w.bad = true;
    if (w.bad) throw std::runtime_error("the lanes of a wave have diverged");
}

inline uint32_t lane_id() { return static_cast<uint32_t>(wave().lane); }

}  // namespace host_wave

inline int __builtin_amdgcn_readlane(int v, uint32_t lane) {
    return static_cast<int>(host_wave::meet(static_cast<uint32_t>(v), 1u)[lane & 63u]);
}

inline int __builtin_amdgcn_readfirstlane(int v) { return static_cast<int>(host_wave::meet(static_cast<uint32_t>(v), 2u)[0]); }

inline uint64_t __ballot(bool v) {
    const uint32_t* all = host_wave::meet(v ? 1u : 0u, 3u);
    uint64_t mask = 0u;
    for (int i = 0; i < 64; ++i) mask |= static_cast<uint64_t>(all[i]) << i;
    return mask;
}

// Moves within rows of 16 lanes by `control` & 15 (0x110 ..), of a row's last lane to the next row (0x142), of lane 31 to
// the upper half (0x143); rows outside the mask and lanes that nothing reaches keep `old`.
inline int __builtin_amdgcn_update_dpp(int old, int v, int control, int row_mask, int, bool) {
    const uint32_t* all = host_wave::meet(static_cast<uint32_t>(v), 4u + static_cast<uint32_t>(control));
    const uint32_t lane = host_wave::lane_id();
    const uint32_t row = lane / 16u;
    if (((row_mask >> row) & 1) == 0) return old;
    if ((control & 0xFF0) == 0x110) {
        const uint32_t by = static_cast<uint32_t>(control & 15);
        return lane % 16u >= by ? static_cast<int>(all[lane - by]) : old;
    }
    if (control == 0x142) return row != 0u ? static_cast<int>(all[16u * row - 1u]) : old;
    if (control == 0x143) return row >= 2u ? static_cast<int>(all[31]) : old;
    abort();
}

inline float __builtin_amdgcn_rcpf(float v) { return 1.0f / v; }
