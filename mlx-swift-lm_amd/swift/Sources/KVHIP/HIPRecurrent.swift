// A gated delta layer's state, and beam search over caches.
import CKVHIP
import Foundation

/// What hybrid models keep in a `MambaCache` (KVCache.swift:1307-1726) beside the KV caches of their attention layers: the short
/// convolution's window [B, W - 1, C] and the delta rule's state [B, Hv, Dv, Dk] in float32.  Not trimmable: keep the old arrays.
public final class HIPGatedDeltaCache<A: HIPArray> {
    public var window: A?, deltaState: A?
    public private(set) var offset = 0
    var stream: UnsafeMutableRawPointer? = nil

    public init() {}
    public var isTrimmable: Bool { false }
    @discardableResult public func trim(_ n: Int) -> Int { 0 }

    /// The short convolution of x [B, L, C] with weight [C, W] behind the window, which moves on.
    public func convolve(_ x: A, weight: A, bias: A? = nil, silu: Bool = true, leftPad: UnsafePointer<Int32>? = nil,
                         lengths: UnsafePointer<Int32>? = nil) -> A {
        let s = x.shape, w = weight.shape[1]
        let out = A.empty(s, dtype: x.kvhipDType)
        let new = window ?? A.empty([s[0], w - 1, s[2]], dtype: x.kvhipDType)
        must(kvhip_short_convolution(x.devicePointer, Int64(s[1] * s[2]), Int64(s[2]), weight.devicePointer, bias?.devicePointer, Int32(s[0]),
                                     Int32(s[1]), Int32(s[2]), Int32(w), x.kvhipDType, silu ? 1 : 0, leftPad, lengths,
                                     window?.devicePointer, new.devicePointer, out.devicePointer, stream))
        window = new
        return out
    }

    /// `gatedDeltaUpdate` (GatedDelta.swift:112): q, k [B, L, Hk, Dk], v [B, L, Hv, Dv], a, b [B, L, Hv]; aLog and dtBias [Hv] in float32.
    public func update(q: A, k: A, v: A, a: A, b: A, aLog: A, dtBias: A, scale: Float? = nil, normEps: Float = 1e-6,
                       leftPad: UnsafePointer<Int32>? = nil, lengths: UnsafePointer<Int32>? = nil) -> A {
        let sk = k.shape, sv = v.shape, f32 = Int32(KVHIP_F32.rawValue)
        let B = sv[0], L = sv[1], Hv = sv[2], Dv = sv[3], Hk = sk[2], Dk = sk[3]
        let out = A.empty(sv, dtype: v.kvhipDType)
        let new = deltaState ?? A.empty([B, Hv, Dv, Dk], dtype: f32)
        var x = kvhip_gated_delta_args()
        (x.q, x.k, x.v) = (UnsafeRawPointer(q.devicePointer), UnsafeRawPointer(k.devicePointer), UnsafeRawPointer(v.devicePointer))
        (x.a, x.b) = (UnsafeRawPointer(a.devicePointer), UnsafeRawPointer(b.devicePointer))
        (x.q_stride_b, x.q_stride_l) = (Int64(L * Hk * Dk), Int64(Hk * Dk))
        (x.k_stride_b, x.k_stride_l) = (x.q_stride_b, x.q_stride_l)
        (x.v_stride_b, x.v_stride_l) = (Int64(L * Hv * Dv), Int64(Hv * Dv))
        (x.a_stride_b, x.a_stride_l) = (Int64(L * Hv), Int64(Hv))
        (x.b_stride_b, x.b_stride_l) = (x.a_stride_b, x.a_stride_l)
        x.a_log = UnsafePointer(aLog.devicePointer.assumingMemoryBound(to: Float.self))
        x.dt_bias = UnsafePointer(dtBias.devicePointer.assumingMemoryBound(to: Float.self))
        (x.left_pad, x.lengths) = (leftPad, lengths)
        x.state_in = deltaState.map { UnsafePointer($0.devicePointer.assumingMemoryBound(to: Float.self)) }
        x.state_out = new.devicePointer.assumingMemoryBound(to: Float.self)
        x.out = out.devicePointer
        (x.B, x.L, x.Hk, x.Hv, x.Dk, x.Dv) = (Int32(B), Int32(L), Int32(Hk), Int32(Hv), Int32(Dk), Int32(Dv))
        (x.dtype, x.gate_dtype) = (v.kvhipDType, a.kvhipDType)
        (x.scale, x.norm_eps) = (scale ?? pow(Float(Dk), -0.5), normEps)
        let need = kvhip_gated_delta_workspace(&x)
        let scratch = need > 0 ? A.empty([(need + 3) / 4], dtype: f32) : nil
        must(kvhip_gated_delta(&x, scratch?.devicePointer, need, stream))
        deltaState = new
        offset += L
        return out
    }

    /// Sequence b becomes what sequence order[b] was.
    public func reorder(order: UnsafePointer<Int32>) {
        let held = [window, deltaState].compactMap { $0 }.filter { $0.shape.allSatisfy { $0 > 0 } }
        guard let rows = held.first?.shape[0] else { return }
        var at: [UnsafeMutableRawPointer?] = held.map { $0.devicePointer }
        var bytes = held.map { a in a.shape.dropFirst().reduce(1, *) * (a.kvhipDType == Int32(KVHIP_F32.rawValue) ? 4 : 2) }
        must(kvhip_reorder_rows(Int32(held.count), &at, &bytes, Int32(rows), order, stream))
    }
}

extension HIPKVCache {
    /// Sequence b of the batch becomes what sequence order[b] was (`beamSelect`'s rows, on the device); the first `shared` positions
    /// are known to be the same.
    public func reorder(order: UnsafePointer<Int32>, shared: Int = 0) {
        must(kvhip_cache_reorder(handle, order, Int64(shared), stream))
    }
}

/// The `count` best continuations of each batch row's beams, logits [B, K, V] and scores [B, K] (float32): best first, into device arrays
/// [B, count]; `rows` is an order for every cache's `reorder` when count is K.
public func beamSelect<A: HIPArray>(logits: A, scores: A?, count: Int, rows: UnsafeMutablePointer<Int32>, tokens: UnsafeMutablePointer<Int32>,
                                    best: UnsafeMutablePointer<Float>, done: UnsafePointer<UInt8>? = nil, padToken: Int = 0,
                                    stream: UnsafeMutableRawPointer? = nil) throws {
    let s = logits.shape
    let need = kvhip_beam_select_workspace(Int32(s[0]), Int32(s[1]), Int32(s[2]), logits.kvhipDType, Int32(count))
    let scratch = A.empty([max((need + 3) / 4, 1)], dtype: Int32(KVHIP_F32.rawValue))
    try check(kvhip_beam_select(logits.devicePointer, Int64(s[2]), Int32(s[0]), Int32(s[1]), Int32(s[2]), logits.kvhipDType,
                                scores.map { UnsafePointer($0.devicePointer.assumingMemoryBound(to: Float.self)) }, done, Int32(count),
                                Int32(padToken), rows, tokens, best, scratch.devicePointer, need, stream))
}
