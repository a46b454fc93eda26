//! Operators built on the k largest values of a row (include/zg_hip_topk.h) for Zigrad's HipDevice: selection, the loss of a
//! student against a teacher's k largest logits, rows to experts and back, the experts' Linear layers.
//!
//! Drop this file next to hip_device.zig.  The reference has no op of these names, so they are functions of a device rather than
//! members of the opspec contract: `hip_topk.topk_fwd(device, .{ .x = ..., ... })`.  Sizes follow from the slices where they can;
//! what the library refuses becomes @panic with its message, as in hip_device.zig.
//!
//! This file cannot be compiled in the build container (no Zig toolchain); the calls' arguments are checked against the header
//! by a static test.
const std = @import("std");
const c = @cImport(@cInclude("zg_hip_topk.h"));
const HipDevice = @import("hip_device.zig");

fn check(rc: c_int) void {
    if (rc != 0) std.debug.panic("zg_hip: {s}", .{std.mem.span(c.zg_hip_last_error())});
}
fn ctx(device: *const HipDevice) *c.zg_hip_ctx {
    return @ptrCast(device.ctx);
}
fn optional(slice: ?[]const f32) ?[*]const f32 {
    return if (slice) |s| s.ptr else null;
}
fn optional_out(slice: ?[]f32) ?[*]f32 {
    return if (slice) |s| s.ptr else null;
}

pub const Selection = struct { x: []const f32, values: []f32, indices: []u64, rows: usize, cols: usize, k: usize };
pub fn topk_fwd(device: *const HipDevice, p: Selection) void {
    std.debug.assert(p.x.len >= p.rows * p.cols and p.values.len >= p.rows * p.k and p.indices.len >= p.rows * p.k);
    check(c.zg_hip_topk_fwd(ctx(device), p.x.ptr, p.values.ptr, @ptrCast(p.indices.ptr), p.rows, p.cols, p.k));
}
pub const SelectionGrad = struct { indices: []const u64, y_g: []const f32, x_g: []f32, rows: usize, cols: usize, k: usize, accumulate: bool = true };
pub fn topk_bwd(device: *const HipDevice, p: SelectionGrad) void {
    std.debug.assert(p.indices.len >= p.rows * p.k and p.y_g.len >= p.rows * p.k and p.x_g.len >= p.rows * p.cols);
    check(c.zg_hip_topk_bwd(ctx(device), @ptrCast(p.indices.ptr), p.y_g.ptr, p.x_g.ptr, p.rows, p.cols, p.k, @intFromBool(p.accumulate)));
}

/// The teacher's k largest logits and their columns, as topk_fwd gives them; row_weights null: the mean.
pub const Distillation = struct {
    logits: []const f32,
    teacher: []const f32,
    indices: []const u64,
    row_weights: ?[]const f32 = null,
    stats: []f32,
    row_loss: []f32 = &.{},
    loss: []f32 = &.{},
    grad: []f32 = &.{},
    rows: usize,
    cols: usize,
    k: usize,
    temperature: f32 = 1,
    accumulate: bool = true,

    fn inputs_fit(p: Distillation) bool {
        return p.logits.len >= p.rows * p.cols and p.teacher.len >= p.rows * p.k and p.indices.len >= p.rows * p.k and
            p.stats.len >= 2 * p.rows and (p.row_weights == null or p.row_weights.?.len >= p.rows);
    }
};
pub fn distill_fwd(device: *const HipDevice, p: Distillation) void {
    std.debug.assert(p.inputs_fit() and p.row_loss.len >= p.rows and p.loss.len >= 1);
    check(c.zg_hip_distill_fwd(ctx(device), p.logits.ptr, p.teacher.ptr, @ptrCast(p.indices.ptr), optional(p.row_weights), p.stats.ptr, p.row_loss.ptr, p.loss.ptr, p.rows, p.cols, p.k, p.temperature));
}
pub fn distill_bwd(device: *const HipDevice, p: Distillation) void {
    std.debug.assert(p.inputs_fit() and p.grad.len >= p.rows * p.cols);
    check(c.zg_hip_distill_bwd(ctx(device), p.logits.ptr, p.teacher.ptr, @ptrCast(p.indices.ptr), optional(p.row_weights), p.stats.ptr, p.grad.ptr, p.rows, p.cols, p.k, p.temperature, @intFromBool(p.accumulate)));
}
/// distill_fwd and the backward of the scalar loss (upstream gradient 1).
pub fn distill_fwd_bwd(device: *const HipDevice, p: Distillation) void {
    std.debug.assert(p.inputs_fit() and p.row_loss.len >= p.rows and p.loss.len >= 1 and p.grad.len >= p.rows * p.cols);
    check(c.zg_hip_distill_fwd_bwd(ctx(device), p.logits.ptr, p.teacher.ptr, @ptrCast(p.indices.ptr), optional(p.row_weights), p.stats.ptr, p.row_loss.ptr, p.loss.ptr, p.grad.ptr, p.rows, p.cols, p.k, p.temperature, @intFromBool(p.accumulate)));
}

/// experts[t * k + j]: where row t goes; offsets and slots: see the header.
pub fn expert_sort(device: *const HipDevice, experts: []const u64, offsets: []u64, slots: []u64, n_experts: usize) void {
    std.debug.assert(offsets.len >= n_experts + 1 and slots.len >= experts.len);
    check(c.zg_hip_expert_sort(ctx(device), @ptrCast(experts.ptr), @ptrCast(offsets.ptr), @ptrCast(slots.ptr), experts.len, n_experts));
}
pub fn expert_dispatch(device: *const HipDevice, x: []const f32, slots: []const u64, y: []f32, n_tokens: usize, k: usize, width: usize) void {
    std.debug.assert(x.len >= n_tokens * width and slots.len >= n_tokens * k and y.len >= n_tokens * k * width);
    check(c.zg_hip_expert_dispatch(ctx(device), x.ptr, @ptrCast(slots.ptr), y.ptr, n_tokens, k, width));
}
pub fn expert_dispatch_bwd(device: *const HipDevice, y_g: []const f32, slots: []const u64, x_g: []f32, n_tokens: usize, k: usize, width: usize, accumulate: bool) void {
    std.debug.assert(y_g.len >= n_tokens * k * width and slots.len >= n_tokens * k and x_g.len >= n_tokens * width);
    check(c.zg_hip_expert_dispatch_bwd(ctx(device), y_g.ptr, @ptrCast(slots.ptr), x_g.ptr, n_tokens, k, width, @intFromBool(accumulate)));
}
pub fn expert_combine(device: *const HipDevice, y: []const f32, slots: []const u64, weights: []const f32, out: []f32, n_tokens: usize, k: usize, width: usize) void {
    std.debug.assert(y.len >= n_tokens * k * width and slots.len >= n_tokens * k and weights.len >= n_tokens * k and out.len >= n_tokens * width);
    check(c.zg_hip_expert_combine(ctx(device), y.ptr, @ptrCast(slots.ptr), weights.ptr, out.ptr, n_tokens, k, width));
}
/// y_g or weights_g may be null, y too when weights_g is.
pub fn expert_combine_bwd(device: *const HipDevice, out_g: []const f32, y: ?[]const f32, slots: []const u64, weights: []const f32, y_g: ?[]f32, weights_g: ?[]f32, n_tokens: usize, k: usize, width: usize) void {
    std.debug.assert(out_g.len >= n_tokens * width and slots.len >= n_tokens * k and weights.len >= n_tokens * k);
    check(c.zg_hip_expert_combine_bwd(ctx(device), out_g.ptr, optional(y), @ptrCast(slots.ptr), weights.ptr, optional_out(y_g), optional_out(weights_g), n_tokens, k, width));
}

pub const ExpertLayer = struct { offsets: []const u64, n_rows: usize, n_experts: usize, fan_in: usize, fan_out: usize };
pub fn expert_linear_fwd(device: *const HipDevice, l: ExpertLayer, x: []const f32, w: []const f32, bias: ?[]const f32, y: []f32, relu: bool) void {
    std.debug.assert(x.len >= l.n_rows * l.fan_in and w.len >= l.n_experts * l.fan_out * l.fan_in and y.len >= l.n_rows * l.fan_out);
    std.debug.assert(l.offsets.len >= l.n_experts + 1);
    check(c.zg_hip_expert_linear_fwd(ctx(device), x.ptr, w.ptr, optional(bias), y.ptr, @ptrCast(l.offsets.ptr), l.n_rows, l.n_experts, l.fan_in, l.fan_out, @intFromBool(relu)));
}
/// gx null: no input gradient; act_in null: no mask; gb null: no bias.
pub fn expert_linear_bwd(device: *const HipDevice, l: ExpertLayer, gy: []const f32, x: []const f32, w: ?[]const f32, act_in: ?[]const f32, gw: []f32, gb: ?[]f32, gx: ?[]f32, accumulate: bool) void {
    std.debug.assert(gy.len >= l.n_rows * l.fan_out and x.len >= l.n_rows * l.fan_in and gw.len >= l.n_experts * l.fan_out * l.fan_in);
    std.debug.assert(l.offsets.len >= l.n_experts + 1);
    check(c.zg_hip_expert_linear_bwd(ctx(device), gy.ptr, x.ptr, optional(w), optional(act_in), gw.ptr, optional_out(gb), optional_out(gx), @ptrCast(l.offsets.ptr), l.n_rows, l.n_experts, l.fan_in, l.fan_out, @intFromBool(accumulate)));
}
