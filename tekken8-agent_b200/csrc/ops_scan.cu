// C entries of the selective scan: argument checks, and what the workspace holds.
#include "ops_scan.cuh"

namespace t8b {
namespace op {
namespace scan {

extern template void launch_forward<float>(const Call&, const ForwardPlan&, int64_t, cudaStream_t);
extern template void launch_forward<bf16>(const Call&, const ForwardPlan&, int64_t, cudaStream_t);
extern template void launch_forward<f16>(const Call&, const ForwardPlan&, int64_t, cudaStream_t);
extern template void launch_backward<float>(const Call&, const BackwardPlan&, float*, float*, float*, cudaStream_t);
extern template void launch_backward<bf16>(const Call&, const BackwardPlan&, float*, float*, float*, cudaStream_t);
extern template void launch_backward<f16>(const Call&, const BackwardPlan&, float*, float*, float*, cudaStream_t);
extern template void launch_step<float>(const Call&, float*, bool, cudaStream_t);
extern template void launch_step<bf16>(const Call&, float*, bool, cudaStream_t);
extern template void launch_step<f16>(const Call&, float*, bool, cudaStream_t);

namespace {

// Where the parts of a workspace start, in floats, each on 256 bytes; `total` of them in all.
struct Room {
    size_t carry = 0, sizes = 0, keep = 0, shared = 0, partial = 0, total = 0;
    void chunks(const t8b_sequences_t& q, int64_t states, int64_t count) {
        if (count <= 1) return;
        const size_t at = static_cast<size_t>(q.sequences) * count;
        carry = take(at * states * q.channels);
        sizes = take(at * q.channels);
        keep = take(at);
    }
    size_t take(size_t floats) {
        const size_t at = total;
        total += round_up(floats, 64);
        return at;
    }
    Room(const t8b_sequences_t& q, int64_t states, const ForwardPlan& plan) { chunks(q, states, plan.chunks); }
    Room(const t8b_sequences_t& q, int64_t groups, int64_t states, const BackwardPlan& plan) {
        chunks(q, states, plan.chunks);
        shared = take(static_cast<size_t>(plan.group_blocks) * groups * q.sequences * q.steps * 2 * states);
        partial = take(static_cast<size_t>(plan.workers) * (states + 2) * q.channels);
    }
};

bool sane(const t8b_sequences_t* q, int64_t groups, int64_t states) {
    return q != nullptr && countable(*q) && q->sequences >= 1 && q->steps >= 1 && groups >= 1 && q->channels % groups == 0 && states >= 1 &&
        states <= kMostStates;
}

// What every call checks, and its inputs' spans.
void check_call(const char* what, const t8b_sequences_t* q, bool step, const t8b_scan_t* scan, Overlaps& o) {
    check_sequences(what, q, step);
    const std::string name(what);
    if (scan == nullptr) raise(T8B_EINVAL, name + ": the scan is null");
    if (!is_type(scan->type)) raise(T8B_EINVAL, name + ": unknown type");
    if (scan->states < 1 || scan->states > kMostStates) raise(T8B_EINVAL, name + ": 1 to 64 states");
    if (scan->groups < 1 || q->channels % scan->groups != 0) raise(T8B_EINVAL, name + ": the groups must divide the channels");
    const size_t size = type_size(scan->type);
    auto track = [&](const char* which, const t8b_track_t& t, int64_t width) {
        check_track((name + " " + which).c_str(), *q, step, t, width, size, false);
        o.input(span_of(*q, step, t, width, size));
    };
    track("u", scan->u, q->channels);
    track("delta", scan->delta, q->channels);
    if (scan->z.data) track("z", scan->z, q->channels);
    for (int64_t apart : {scan->b_group, scan->c_group}) {
        if (apart < 0 || apart > kMostElements / scan->groups) raise(T8B_EINVAL, name + ": a group stride is out of range");
    }
    track("b", scan->b, (scan->groups - 1) * scan->b_group + scan->states);
    track("c", scan->c, (scan->groups - 1) * scan->c_group + scan->states);
    if (scan->a == nullptr) raise(T8B_EINVAL, name + ": a is null");
    for (const float* p : {scan->a, scan->d, scan->delta_bias}) {
        check_elements(what, p, sizeof(float));
        o.input(span_of(p, q->channels * (p == scan->a ? scan->states : 1), sizeof(float)));
    }
    if (!step) {
        check_elements(what, scan->state, sizeof(float));
        o.input(span_of(scan->state, q->sequences * q->channels * scan->states, sizeof(float)));
    }
    o.input(span_of(scan->a, q->channels * scan->states, sizeof(float)));
}
Call call_of(const t8b_sequences_t& q, const t8b_scan_t& scan) {
    Call a{};
    a.q = Sequences(q);
    a.u = Track<void>(scan.u);
    a.delta = Track<void>(scan.delta);
    a.z = Track<void>(scan.z);
    a.b = Track<void>(scan.b);
    a.c = Track<void>(scan.c);
    a.b_group = scan.b_group;
    a.c_group = scan.c_group;
    a.a = scan.a;
    a.d = scan.d;
    a.delta_bias = scan.delta_bias;
    a.state = scan.state;
    a.groups = static_cast<int>(scan.groups);
    a.per = static_cast<int>(q.channels / scan.groups);
    a.states = static_cast<int>(scan.states);
    a.softplus = scan.softplus;
    return a;
}
// Whether `count` neighbouring channels of every row of a track may be accessed at once.
bool together(const t8b_sequences_t& q, const t8b_scan_t& scan, const t8b_track_t& t, int64_t count) {
    const size_t size = type_size(scan.type);
    return t.data == nullptr || (q.channels / scan.groups % count == 0 && rows_aligned(q, false, t, size, count * size));
}
void check_room(const char* what, const void* workspace, size_t given, size_t needed) {
    if (needed && (workspace == nullptr || given < needed || !aligned(workspace, 256))) {
        raise(T8B_EINVAL, std::string(what) + ": the workspace is missing, unaligned or smaller than t8b_selective_scan_workspace");
    }
}
void check_grid(const char* what, int64_t blocks) {
    if (blocks > std::numeric_limits<int32_t>::max()) raise(T8B_EINVAL, std::string(what) + ": too many elements for one call");
}

}  // namespace
}  // namespace scan
}  // namespace op
}  // namespace t8b

using namespace t8b;
using namespace t8b::op;
using namespace t8b::op::scan;

extern "C" size_t t8b_selective_scan_saved(const t8b_sequences_t* q, int64_t groups, int64_t states) {
    if (!sane(q, groups, states)) return 0;
    return static_cast<size_t>(q->sequences) * tiles_of(q->steps) * states * q->channels;
}

extern "C" size_t t8b_selective_scan_workspace(const t8b_sequences_t* q, int64_t groups, int64_t states, int backward) {
    if (!sane(q, groups, states)) return 0;
    const Room room = backward ? Room(*q, groups, states, BackwardPlan(*q, groups, states)) : Room(*q, states, ForwardPlan(*q, groups, states));
    return room.total * sizeof(float);
}

extern "C" int t8b_selective_scan_forward(const t8b_sequences_t* q, const t8b_scan_t* scan, t8b_track_t y, float* final_state,
                                          float* saved, void* workspace, size_t workspace_bytes, void* stream) {
    return guarded([&] {
        Overlaps o{"selective scan"};
        check_call("selective scan", q, false, scan, o);
        const size_t size = type_size(scan->type);
        check_track("selective scan y", *q, false, y, q->channels, size, true);
        for (const float* p : {final_state, saved}) check_elements("selective scan states", p, sizeof(float));
        if (q->sequences == 0) return;
        const int64_t held = q->sequences * q->channels * scan->states;
        o.output(span_of(*q, false, y, q->channels, size));
        o.output(span_of(final_state, held, sizeof(float)));
        o.output(span_of(saved, t8b_selective_scan_saved(q, scan->groups, scan->states), sizeof(float)));
        const ForwardPlan plan(*q, scan->groups, scan->states);
        check_grid("selective scan", std::max(plan.blocks, (held + 255) / 256));
        const Room room(*q, scan->states, plan);
        check_room("selective scan", workspace, workspace_bytes, room.total * sizeof(float));
        Call a = call_of(*q, *scan);
        a.y = Track<void>(y);
        a.final_state = final_state;
        a.saved = saved;
        a.wide = 1;
        for (const t8b_track_t* t : {&scan->u, &scan->delta, &scan->z, static_cast<const t8b_track_t*>(&y)}) a.wide &= together(*q, *scan, *t, 16 / size);
        float* w = static_cast<float*>(workspace);
        a.carry = w + room.carry;
        a.sizes = w + room.sizes;
        a.keep = w + room.keep;
        with_type(scan->type, [&](auto element) { launch_forward<decltype(element)>(a, plan, scan->states, static_cast<cudaStream_t>(stream)); });
        check(cudaGetLastError(), "selective scan launch");
    });
}

extern "C" int t8b_selective_scan_backward(const t8b_sequences_t* q, const t8b_scan_t* scan, t8b_track_t dy, const float* saved,
                                           const float* final_gradient, const t8b_scan_gradients_t* gradients, void* workspace,
                                           size_t workspace_bytes, void* stream) {
    return guarded([&] {
        Overlaps o{"selective scan"};
        check_call("selective scan", q, false, scan, o);
        if (gradients == nullptr || gradients->da == nullptr) raise(T8B_EINVAL, "selective scan: the gradients are null");
        const t8b_scan_gradients_t& g = *gradients;
        const size_t size = type_size(scan->type);
        const int64_t held = q->sequences * q->channels * scan->states;
        check_track("selective scan dy", *q, false, dy, q->channels, size, false);
        o.input(span_of(*q, false, dy, q->channels, size));
        for (const float* p : {saved, final_gradient, static_cast<const float*>(g.da), static_cast<const float*>(g.dd),
                               static_cast<const float*>(g.ddelta_bias), static_cast<const float*>(g.dstate)}) {
            check_elements("selective scan", p, sizeof(float));
        }
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        if (q->sequences == 0 || q->steps == 0) {
            check(cudaMemsetAsync(g.da, 0, sizeof(float) * q->channels * scan->states, st), "clear da");
            if (g.dd) check(cudaMemsetAsync(g.dd, 0, sizeof(float) * q->channels, st), "clear dd");
            if (g.ddelta_bias) check(cudaMemsetAsync(g.ddelta_bias, 0, sizeof(float) * q->channels, st), "clear ddelta_bias");
            if (g.dstate && held) {
                if (final_gradient) {
                    check(cudaMemcpyAsync(g.dstate, final_gradient, sizeof(float) * held, cudaMemcpyDeviceToDevice, st), "dstate");
                } else {
                    check(cudaMemsetAsync(g.dstate, 0, sizeof(float) * held, st), "clear dstate");
                }
            }
            return;
        }
        if (saved == nullptr) raise(T8B_EINVAL, "selective scan: what the forward pass saved is null");
        o.input(span_of(saved, t8b_selective_scan_saved(q, scan->groups, scan->states), sizeof(float)));
        o.input(span_of(final_gradient, held, sizeof(float)));
        auto track = [&](const char* which, const t8b_track_t& t, int64_t width) {
            check_track(which, *q, false, t, width, size, true);
            o.output(span_of(*q, false, t, width, size));
        };
        track("selective scan du", g.du, q->channels);
        track("selective scan ddelta", g.ddelta, q->channels);
        if (g.dz.data) {
            if (!scan->z.data) raise(T8B_EINVAL, "selective scan: dz without z");
            track("selective scan dz", g.dz, q->channels);
        }
        for (int64_t apart : {g.db_group, g.dc_group}) {
            if (scan->groups > 1 && (apart < scan->states || apart > kMostElements / scan->groups)) {
                raise(T8B_EINVAL, "selective scan: a gradient's group stride is out of range");
            }
        }
        track("selective scan db", g.db, (scan->groups - 1) * g.db_group + scan->states);
        track("selective scan dc", g.dc, (scan->groups - 1) * g.dc_group + scan->states);
        o.output(span_of(g.da, q->channels * scan->states, sizeof(float)));
        o.output(span_of(g.dd, q->channels, sizeof(float)));
        o.output(span_of(g.ddelta_bias, q->channels, sizeof(float)));
        o.output(span_of(g.dstate, held, sizeof(float)));
        const BackwardPlan plan(*q, scan->groups, scan->states);
        check_grid("selective scan", std::max({q->sequences * plan.chunks * scan->groups * plan.end_blocks, (held + 255) / 256,
                                               (scan->groups * q->sequences * q->steps * 2 * scan->states + 255) / 256}));
        const Room room(*q, scan->groups, scan->states, plan);
        check_room("selective scan", workspace, workspace_bytes, room.total * sizeof(float));
        Call a = call_of(*q, *scan);
        a.dy = Track<void>(dy);
        a.saved = const_cast<float*>(saved);
        // four channels of a row (or two, or one) at once in the backward pass's elementwise part
        const int width = scan->states <= 16 ? 4 : scan->states <= 32 ? 2 : 1;
        a.paired = 1;
        for (const t8b_track_t* t : {&scan->u, &scan->delta, &scan->z, static_cast<const t8b_track_t*>(&dy), &g.du, &g.ddelta, &g.dz}) {
            a.paired &= together(*q, *scan, *t, width);
        }
        a.saved_paired = q->channels / scan->groups % 2 == 0 && aligned(saved, 8);
        a.final_gradient = final_gradient;
        a.du = Track<void>(g.du);
        a.ddelta = Track<void>(g.ddelta);
        a.dz = Track<void>(g.dz);
        a.db = Track<void>(g.db);
        a.dc = Track<void>(g.dc);
        a.db_group = g.db_group;
        a.dc_group = g.dc_group;
        a.dstate = g.dstate;
        float* w = static_cast<float*>(workspace);
        a.carry = w + room.carry;
        a.sizes = w + room.sizes;
        a.keep = w + room.keep;
        a.shared = w + room.shared;
        a.partial = w + room.partial;
        with_type(scan->type, [&](auto element) { launch_backward<decltype(element)>(a, plan, g.da, g.dd, g.ddelta_bias, st); });
        check(cudaGetLastError(), "selective scan launch");
    });
}

extern "C" int t8b_selective_scan_step(const t8b_sequences_t* q, const t8b_scan_t* scan, float* state, t8b_track_t y, void* stream) {
    return guarded([&] {
        Overlaps o{"selective scan step"};
        check_call("selective scan step", q, true, scan, o);
        const size_t size = type_size(scan->type);
        check_track("selective scan step y", *q, true, y, q->channels, size, true);
        check_elements("selective scan step state", state, sizeof(float));
        if (q->sequences == 0) return;
        if (state == nullptr) raise(T8B_EINVAL, "selective scan step: state is null");
        o.output(span_of(*q, true, y, q->channels, size));
        o.output(span_of(state, q->sequences * q->channels * scan->states, sizeof(float)));
        Call a = call_of(*q, *scan);
        a.y = Track<void>(y);
        const bool wide = scan->states % 4 == 0 && aligned(state, 16) && aligned(scan->a, 16);
        with_type(scan->type, [&](auto element) { launch_step<decltype(element)>(a, state, wide, static_cast<cudaStream_t>(stream)); });
        check(cudaGetLastError(), "selective scan step launch");
    });
}
