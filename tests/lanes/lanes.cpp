// Runs a kernel's workgroups on the CPU, one after the other, each lane a coroutine
// with a stack of its own (x86-64).  A lane goes on until it needs the others of its
// wave or workgroup; a wave of which some lanes wait for the wave and some for the
// workgroup ends the process.
#include <hip/hip_runtime.h>
#include <stdarg.h>
#include <stdio.h>
#include <stdlib.h>
#include <sys/mman.h>

#include <vector>

extern "C" void lanes_switch(void** from, void* to);
asm(R"(
.text
.globl lanes_switch
lanes_switch:
    pushq %rbp
    pushq %rbx
    pushq %r12
    pushq %r13
    pushq %r14
    pushq %r15
    movq %rsp, (%rdi)
    movq %rsi, %rsp
    popq %r15
    popq %r14
    popq %r13
    popq %r12
    popq %rbx
    popq %rbp
    ret
)");

namespace lanes {

dim3 thread, block, grid;
bool skip_products = false;

namespace {
enum State { kRuns, kWantsWave, kWantsBlock, kDone };
struct Lane {
    void* stack_pointer;
    unsigned char* stack = nullptr;
    State state;
    int turn;
};
constexpr size_t kStack = 512 << 10;
constexpr int kMost = 1024;
Lane all[kMost];
Values values[kMost / 64][2];
uint64_t still[kMost / 64];
void* scheduler;
const void* current_arguments;
const std::function<void()>* current_kernel;

void leave(State state) {
    Lane& l = all[thread.x];
    l.state = state;
    lanes_switch(&l.stack_pointer, scheduler);
}
void enter() {
    (*current_kernel)();
    leave(kDone);
}

int count_of(int from, int to, State state) {
    int n = 0;
    for (int i = from; i < to; ++i) n += all[i].state == state;
    return n;
}

void run_block(int count) {
    for (int i = 0; i < count; ++i) {
        Lane& l = all[i];
        if (!l.stack)
            l.stack = (unsigned char*)mmap(nullptr, kStack, PROT_READ | PROT_WRITE, MAP_PRIVATE | MAP_ANONYMOUS, -1, 0);
        void** top = (void**)(l.stack + kStack);
        *--top = nullptr;
        *--top = (void*)enter;
        for (int saved = 0; saved < 6; ++saved) *--top = nullptr;
        l.stack_pointer = top;
        l.state = kRuns;
        l.turn = 0;
    }
    for (int w = 0; w < count / 64; ++w) still[w] = ~uint64_t(0);
    while (count_of(0, count, kDone) < count) {
        for (int begin = 0; begin < count; begin += 64) {
            const int end = begin + 64;
            while (count_of(begin, end, kRuns)) {
                for (int i = begin; i < end; ++i) {
                    if (all[i].state != kRuns) continue;
                    thread = dim3((unsigned)i);
                    lanes_switch(&scheduler, all[i].stack_pointer);
                }
                for (int i = begin; i < end; ++i)
                    if (all[i].state == kDone) still[begin / 64] &= ~(uint64_t(1) << (i - begin));
                if (!count_of(begin, end, kWantsWave)) break;
                if (count_of(begin, end, kWantsBlock)) fail("a wave's lanes wait at different places");
                for (int i = begin; i < end; ++i)
                    if (all[i].state == kWantsWave) all[i].state = kRuns;
            }
        }
        for (int i = 0; i < count; ++i)
            if (all[i].state == kWantsBlock) all[i].state = kRuns;
    }
}
}  // namespace

uint64_t alive() { return still[thread.x / 64]; }
const void* arguments() { return current_arguments; }
void wave_sync() { leave(kWantsWave); }
void block_sync() { leave(kWantsBlock); }

const Values& exchange(const void* value, size_t bytes) {
    Lane& l = all[thread.x];
    Values& v = values[thread.x / 64][l.turn];
    l.turn ^= 1;
    memcpy(v.of[lane()], value, bytes);
    wave_sync();
    return v;
}

void fail(const char* what) {
    fprintf(stderr, "lanes: %s (workgroup %u, thread %u)\n", what, block.x, thread.x);
    abort();
}

void launch(dim3 blocks, dim3 threads, const void* arguments, const std::function<void()>& kernel) {
    if (threads.x % 64 || threads.x > kMost) fail("workgroup size");
    current_arguments = arguments, current_kernel = &kernel, grid = blocks;
    for (unsigned b = 0; b < blocks.x; ++b) {
        block = dim3(b);
        run_block((int)threads.x);
    }
}

}  // namespace lanes

// The library's errors.
namespace w4g64 {
char message[512];
int set_error(int status, const char* format, ...) {
    va_list list;
    va_start(list, format);
    vsnprintf(message, sizeof(message), format, list);
    va_end(list);
    return status;
}
int clear_error() { return 0; }
}  // namespace w4g64

extern "C" const char* lanes_error() { return w4g64::message; }
extern "C" void lanes_skip_products(int skip) { lanes::skip_products = skip != 0; }
