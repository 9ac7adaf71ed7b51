// Whether what a call writes shares memory with what it reads.  Plain host code, so that it can be tested without a device.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include <initializer_list>

// Pieces of `width` bytes in memory: `n` of them `step` bytes apart, and that `groups` times, `group_step` apart.
struct Pieces {
    const void *at;
    size_t width;
    long long n, step, groups, group_step;
};

// Whether a piece of `read` shares memory with one of `written`, whose pieces lie apart, those of a group before those of the next.
// Costs a few comparisons where the two lie apart as wholes, else a look at every piece that is read, or, for the same steps, at every
// distance between the pieces of two groups.
inline bool pieces_overlap(const Pieces &written, const Pieces &read) {
    typedef __int128 wide;   // (any stride is a legal one for what is read)
    Pieces w = written, r = read;
    for (Pieces *p : {&w, &r}) {   // a step that is not taken does not count
        if (p->n < 2) p->n = 1, p->step = 0;
        if (p->groups < 2) p->groups = 1, p->group_step = 0;
    }
    auto size = [](const Pieces &p) { return (wide)(p.n - 1) * p.step + (wide)(p.groups - 1) * p.group_step + p.width; };
    const wide apart = (wide)(uintptr_t)r.at - (wide)(uintptr_t)w.at, w_size = size(w);   // from the first piece written to the first read
    if (apart >= w_size || -apart >= size(r)) return false;
    auto meet = [&](wide distance) { return distance < (wide)w.width && -distance < (wide)r.width; };   // of a piece read from one written
    // the number from 0 to n - 1 whose multiple of step is the last one at or below d (0 where none is)
    auto index = [](wide d, long long step, long long n) { return step <= 0 || d < 0 ? 0 : d / step >= n ? n - 1 : (long long)(d / step); };
    if (w.n == r.n && w.groups == r.groups && w.step == r.step && w.group_step == r.group_step) {
        for (long long j = 1 - w.n; j < w.n; ++j) {
            const wide d = apart + (wide)j * w.step;
            // the multiples of group_step on either side of d
            const long long k = index(d < 0 ? -d : d, w.group_step, w.groups);
            for (long long i = k; i <= k + 1 && i < w.groups; ++i)
                if (meet(d < 0 ? d + (wide)i * w.group_step : d - (wide)i * w.group_step)) return true;
        }
        return false;
    }
    if (r.step == 0) r.n = 1;
    if (r.group_step == 0) r.groups = 1;
    for (long long g = 0; g < r.groups; ++g)
        for (long long j = 0; j < r.n; ++j) {
            const wide d = apart + (wide)g * r.group_step + (wide)j * r.step;   // from the first piece written
            if (d >= w_size || -d >= (wide)r.width) continue;
            // groups that begin before the piece ends, from the one it begins in: they lie apart, so a piece that passes one's end meets the next
            for (long long k = index(d, w.group_step, w.groups); k < w.groups && (wide)k * w.group_step < d + (wide)r.width; ++k) {
                const wide in = d - (wide)k * w.group_step;
                for (long long i = index(in, w.step, w.n); i < w.n && (wide)i * w.step < in + (wide)r.width; ++i)
                    if (meet(in - (wide)i * w.step)) return true;
            }
        }
    return false;
}
